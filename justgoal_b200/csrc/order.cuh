// Token order of an MoE layer for training: the (token, pick) pairs sorted by expert, token rows into that order and
// back, and their gradients.  T tokens with K picks each, pair i = t K + k, El local experts, row r of a pair.
//
//   sort      expert_row0[e] = sum over f < e of ceil(count_f / align) align; the pairs of an expert stand in ascending
//             pair order (a stable counting sort); row_pair[r] = i or -1, pair_row[i] = r or -1
//   permute   rows[r] = x[t]                        restore   rows[r] = q[t] * scale[., t] (activations kept in 8 bits)
//   combine   out[t] = sum_k w[t, k] rows[r(t, k)]  permute's gradient is the same sum with weights of one
//   combine's gradient   d_rows[r] = w d_out[t],    d_w[t, k] = sum_h d_out[t, h] rows[r, h]
//
// Sums are fp32 in ascending k, rounded once.  Rows of a segment's padding are zeros (a weight gradient sums over whole
// segments); rows behind the last segment are neither read nor written.  Every index that is read from a table is checked
// against its range before it is used, so that tables that do not belong to the call cannot lead outside the buffers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace b200moe {

constexpr int ORDER_MAX_LOCAL = 512;
constexpr int ORDER_MAX_PICKS = 8;

// ---------------------------------------------------------------- element types
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};

// N elements (a multiple of eight) at a 32-byte aligned address (16-byte where N elements are 16 bytes) <-> fp32 values
template <typename T, int N>
__device__ __forceinline__ void load_elems(const T* src, float* v) {
    constexpr int W = N * (int)sizeof(T) / 4;
    uint32_t w[W];
    if constexpr (W == 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(src);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 8) ld_global_v8(reinterpret_cast<const uint32_t*>(src) + i, w + i);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) { const float2 f = Elem<T>::unpack(w[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_elems(T* dst, const float* v) {
    constexpr int W = N * (int)sizeof(T) / 4;
    uint32_t w[W];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = Elem<T>::pack(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (W == 4) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 8)
            st_global_v8(reinterpret_cast<uint32_t*>(dst) + i, w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5], w[i + 6], w[i + 7]);
    }
}

// ---------------------------------------------------------------- sort
constexpr int SORT_THREADS = 1024;
constexpr int SORT_SLICE = 2 * SORT_THREADS;      // pairs of a CTA where several share the work
constexpr int SORT_ONE = 4 * SORT_THREADS;        // most pairs that one CTA sorts alone

struct SortParams {
    const int32_t* topk_idx;      // [n], n = T K
    int n, num_local, local_offset, align, max_rows;
    int* slices;                  // [CTAs][num_local] histogram per slice; several CTAs only
    int32_t *expert_row0, *row_pair, *pair_row;
};

// First row of every expert from the counts, by one warp: lane l owns the experts [l per, (l + 1) per).
__device__ __forceinline__ void sort_scan(const int* count, int num_local, int align, int* row0, int lane) {
    const int per = (num_local + 31) / 32, e0 = lane * per;
    int sum = 0;
    for (int e = e0; e < min(e0 + per, num_local); ++e) sum += (count[e] + align - 1) & -align;
    int upto = sum;
    for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, off);
        if (lane >= off) upto += v;
    }
    int r = upto - sum;
    for (int e = e0; e < min(e0 + per, num_local); ++e) { row0[e] = r; r += (count[e] + align - 1) & -align; }
    if (lane == 31) row0[num_local] = upto;
}

// Places the pairs [begin, end), 1024 at a time: next[e] = row of the expert's next pair, moved on by the pairs placed.
// A pair's rank among the pairs of its expert: match + popcount inside its warp, a prefix over the 32 warps.
__device__ __forceinline__ void sort_place(const SortParams& p, int begin, int end, int* next, uint16_t (*wcnt)[ORDER_MAX_LOCAL + 2]) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, El = p.num_local;
    const unsigned FULL = 0xFFFFFFFFu;
    for (int c = begin; c < end; c += SORT_THREADS) {
        for (int e = lane; e < El; e += 32) wcnt[warp][e] = 0;
        __syncwarp();
        const int i = c + tid;
        const int le = i < end ? __ldg(p.topk_idx + i) - p.local_offset : -1;
        const bool local = le >= 0 && le < El;
        const unsigned same = __match_any_sync(FULL, local ? le : -1 - lane);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (local && rank == 0) wcnt[warp][le] = (uint16_t)__popc(same);
        __syncthreads();
        for (int e = tid; e < El; e += SORT_THREADS) {
            int r = 0;
#pragma unroll 8
            for (int w = 0; w < 32; ++w) { const int v = wcnt[w][e]; wcnt[w][e] = (uint16_t)r; r += v; }
            wcnt[32][e] = (uint16_t)r;
        }
        __syncthreads();
        if (i < end) {
            int r = local ? next[le] + wcnt[warp][le] + rank : -1;
            if (r >= p.max_rows) r = -1;
            p.pair_row[i] = r;
            if (r >= 0) p.row_pair[r] = i;
        }
        __syncthreads();
        for (int e = tid; e < El; e += SORT_THREADS) next[e] += wcnt[32][e];
    }
}

// One CTA for everything: counts, scan, places.
__global__ void __launch_bounds__(SORT_THREADS) sort_one_kernel(const SortParams p) {
    __shared__ int s_count[ORDER_MAX_LOCAL], s_next[ORDER_MAX_LOCAL + 1];
    __shared__ uint16_t s_wcnt[33][ORDER_MAX_LOCAL + 2];
    const int tid = threadIdx.x;
    for (int e = tid; e < p.num_local; e += SORT_THREADS) s_count[e] = 0;
    pdl_wait();
    pdl_launch();
    __syncthreads();
    for (int i = tid; i < p.n; i += SORT_THREADS) {
        const int le = __ldg(p.topk_idx + i) - p.local_offset;
        if (le >= 0 && le < p.num_local) atomicAdd(s_count + le, 1);
    }
    for (int r = tid; r < p.max_rows; r += SORT_THREADS) p.row_pair[r] = -1;
    __syncthreads();
    if (tid < 32) sort_scan(s_count, p.num_local, p.align, s_next, tid);
    __syncthreads();
    for (int e = tid; e <= p.num_local; e += SORT_THREADS) p.expert_row0[e] = min(s_next[e], p.max_rows);
    __syncthreads();
    sort_place(p, 0, p.n, s_next, s_wcnt);
}

// Several CTAs, first kernel: the slice's histogram; row_pair is cleared for the second one.
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortParams p) {
    __shared__ int s_count[ORDER_MAX_LOCAL];
    const int tid = threadIdx.x;
    for (int e = tid; e < p.num_local; e += SORT_THREADS) s_count[e] = 0;
    pdl_wait();
    pdl_launch();
    __syncthreads();
    const int begin = blockIdx.x * SORT_SLICE, end = min(p.n, begin + SORT_SLICE);
    for (int i = begin + tid; i < end; i += SORT_THREADS) {
        const int le = __ldg(p.topk_idx + i) - p.local_offset;
        if (le >= 0 && le < p.num_local) atomicAdd(s_count + le, 1);
    }
    for (int r = blockIdx.x * SORT_THREADS + tid; r < p.max_rows; r += gridDim.x * SORT_THREADS) p.row_pair[r] = -1;
    __syncthreads();
    for (int e = tid; e < p.num_local; e += SORT_THREADS) p.slices[(size_t)blockIdx.x * p.num_local + e] = s_count[e];
}

// Second kernel: every CTA sums the histograms (all of them: the first rows; those before its own: where its pairs start
// inside a segment) and places its slice.  No CTA waits for another.
__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(const SortParams p) {
    __shared__ int s_count[ORDER_MAX_LOCAL], s_before[ORDER_MAX_LOCAL], s_next[ORDER_MAX_LOCAL + 1];
    __shared__ uint16_t s_wcnt[33][ORDER_MAX_LOCAL + 2];
    const int tid = threadIdx.x, El = p.num_local, c = blockIdx.x;
    for (int e = tid; e < El; e += SORT_THREADS) { s_count[e] = 0; s_before[e] = 0; }
    pdl_wait();
    pdl_launch();
    __syncthreads();
    int width = 32;                                   // threads of one row of the table
    while (width < El) width <<= 1;
    const int e = tid & (width - 1);
    if (e < El) {
        int total = 0, before = 0;
#pragma unroll 4
        for (int s = tid / width; s < (int)gridDim.x; s += SORT_THREADS / width) {
            const int v = p.slices[(size_t)s * El + e];
            total += v;
            if (s < c) before += v;
        }
        atomicAdd(s_count + e, total);
        atomicAdd(s_before + e, before);
    }
    __syncthreads();
    if (tid < 32) sort_scan(s_count, El, p.align, s_next, tid);
    __syncthreads();
    if (c == 0)
        for (int k = tid; k <= El; k += SORT_THREADS) p.expert_row0[k] = min(s_next[k], p.max_rows);
    __syncthreads();
    for (int k = tid; k < El; k += SORT_THREADS) s_next[k] += s_before[k];
    __syncthreads();
    const int begin = c * SORT_SLICE;
    sort_place(p, begin, min(p.n, begin + SORT_SLICE), s_next, s_wcnt);
}

// ---------------------------------------------------------------- rows into expert order
struct OrderParams {
    const int32_t* expert_row0;   // [num_local + 1]
    const int32_t* row_pair;      // [num_rows]
    const int32_t* pair_row;      // [T, top_k]
    int T, top_k, num_local, num_rows;
};

// Zeros into the padding rows of the segments, `units` of 32 bytes each: a warp looks at 32 rows at a time.
__device__ __forceinline__ void zero_padding(const OrderParams& o, char* rows, int units, int warp, int warps) {
    const int lane = threadIdx.x & 31;
    const int used = min(__ldg(o.expert_row0 + o.num_local), o.num_rows);
    for (int r0 = warp * 32; r0 < used; r0 += warps * 32) {
        const int pair = r0 + lane < used ? __ldg(o.row_pair + r0 + lane) : 0;
        unsigned empty = __ballot_sync(0xFFFFFFFFu, pair < 0);
        while (empty) {
            const int r = r0 + __ffs(empty) - 1;
            empty &= empty - 1;
            char* dst = rows + (size_t)r * units * 32;
            for (int u = lane; u < units; u += 32) st_global_v8(dst + (size_t)u * 32, 0, 0, 0, 0, 0, 0, 0, 0);
        }
    }
}

// rows[r] = x[t] for the token's rows: a warp takes a token (and one of gridDim.y parts of its columns), reads each 32
// bytes once and stores them up to top_k times.
constexpr int PERMUTE_FLIGHT = 4;
__global__ void __launch_bounds__(256) permute_rows_kernel(const OrderParams o, const char* __restrict__ x, char* __restrict__ rows, int units) {
    const int lane = threadIdx.x & 31;
    const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, warps = (gridDim.x * blockDim.x) >> 5;
    const int per = (units + gridDim.y - 1) / gridDim.y, u_lo = blockIdx.y * per, u_hi = min(units, u_lo + per);
    pdl_wait();
    for (int t = warp; t < o.T; t += warps) {
        int r = -1;
        if (lane < o.top_k) {
            r = __ldg(o.pair_row + (size_t)t * o.top_k + lane);
            if (r >= o.num_rows) r = -1;
        }
        const unsigned have = __ballot_sync(0xFFFFFFFFu, r >= 0);
        const char* src = x + (size_t)t * units * 32;
        for (int u0 = u_lo + lane; u0 - lane < u_hi; u0 += 32 * PERMUTE_FLIGHT) {
            uint32_t v[PERMUTE_FLIGHT][8];
#pragma unroll
            for (int q = 0; q < PERMUTE_FLIGHT; ++q)
                if (have && u0 + 32 * q < u_hi) ld_global_v8(src + (size_t)(u0 + 32 * q) * 32, v[q]);
            for (unsigned todo = have; todo; todo &= todo - 1) {
                char* dst = rows + (size_t)__shfl_sync(0xFFFFFFFFu, r, __ffs(todo) - 1) * units * 32;
#pragma unroll
                for (int q = 0; q < PERMUTE_FLIGHT; ++q)
                    if (u0 + 32 * q < u_hi)
                        st_global_v8(dst + (size_t)(u0 + 32 * q) * 32, v[q][0], v[q][1], v[q][2], v[q][3], v[q][4], v[q][5], v[q][6], v[q][7]);
            }
        }
    }
    pdl_launch();
    if (blockIdx.y == 0) zero_padding(o, rows, units, warp, warps);
}

// 16 e4m3 values times their scale
__device__ __forceinline__ void restore16(const uint4& q, float s, float* v) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = e4m3x2_to_f32x2((uint16_t)w[i]), b = e4m3x2_to_f32x2((uint16_t)(w[i] >> 16));
        v[4 * i] = a.x * s; v[4 * i + 1] = a.y * s; v[4 * i + 2] = b.x * s; v[4 * i + 3] = b.y * s;
    }
}

// rows[r] = q[t] * scale, like permute_rows_kernel with 16 columns per lane and step.  Without an order (pair_row null)
// row t is token t.
template <typename T>
__global__ void __launch_bounds__(256) restore_rows_kernel(const OrderParams o, const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                           T* __restrict__ rows, int H) {
    const int lane = threadIdx.x & 31;
    const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, warps = (gridDim.x * blockDim.x) >> 5;
    const int units = H >> 4;
    const int per = (units + gridDim.y - 1) / gridDim.y, u_lo = blockIdx.y * per, u_hi = min(units, u_lo + per);
    pdl_wait();
    for (int t = warp; t < o.T; t += warps) {
        int r = -1;
        if (!o.pair_row) {
            if (lane == 0) r = t;
        } else if (lane < o.top_k) {
            r = __ldg(o.pair_row + (size_t)t * o.top_k + lane);
            if (r >= o.num_rows) r = -1;
        }
        const unsigned have = __ballot_sync(0xFFFFFFFFu, r >= 0);
        if (!have) continue;
        for (int u0 = u_lo; u0 < u_hi; u0 += 32) {
            const int u = u0 + lane;
            float v[16];
            if (u < u_hi) {
                const uint4 b = __ldg(reinterpret_cast<const uint4*>(q + (size_t)t * H) + u);
                restore16(b, __ldg(scale + (size_t)(u >> 3) * o.T + t), v);
            }
            for (unsigned todo = have; todo; todo &= todo - 1) {
                T* dst = rows + (size_t)__shfl_sync(0xFFFFFFFFu, r, __ffs(todo) - 1) * H;
                if (u < u_hi) store_elems<T, 16>(dst + u * 16, v);
            }
        }
    }
    pdl_launch();
    if (o.pair_row && blockIdx.y == 0) zero_padding(o, reinterpret_cast<char*>(rows), H * (int)sizeof(T) / 32, warp, warps);
}

// ---------------------------------------------------------------- rows back to their tokens
// out[t] = sum_k w[t, k] rows[r(t, k)], w null: ones.  A warp takes a token (and one of gridDim.y parts of its columns); the
// loads of up to eight rows are in flight together.
template <typename T>
__global__ void __launch_bounds__(256) combine_rows_kernel(const OrderParams o, const T* __restrict__ rows, const float* __restrict__ w,
                                                           T* __restrict__ out, int H) {
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, warps = (gridDim.x * blockDim.x) >> 5;
    const int units = H / V;
    const int per = (units + gridDim.y - 1) / gridDim.y, u_lo = blockIdx.y * per, u_hi = min(units, u_lo + per);
    pdl_wait();
    for (int t = warp; t < o.T; t += warps) {
        int r = -1;
        float wt = 1.f;
        if (lane < o.top_k) {
            r = __ldg(o.pair_row + (size_t)t * o.top_k + lane);
            if (r >= o.num_rows) r = -1;
            if (w) wt = __ldg(w + (size_t)t * o.top_k + lane);
        }
        for (int u0 = u_lo; u0 < u_hi; u0 += 32) {
            const int u = u0 + lane;
            uint4 v[ORDER_MAX_PICKS];
#pragma unroll
            for (int k = 0; k < ORDER_MAX_PICKS; ++k) {
                const int rk = __shfl_sync(0xFFFFFFFFu, r, k);
                if (rk >= 0 && u < u_hi) v[k] = __ldcs(reinterpret_cast<const uint4*>(rows + (size_t)rk * H) + u);
            }
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
            for (int k = 0; k < ORDER_MAX_PICKS; ++k) {
                const int rk = __shfl_sync(0xFFFFFFFFu, r, k);
                const float wk = __shfl_sync(0xFFFFFFFFu, wt, k);
                if (rk >= 0 && u < u_hi) {
                    const uint32_t b[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (sizeof(T) == 4) {
                            acc[i] = fmaf(wk, __uint_as_float(b[i]), acc[i]);
                        } else {
                            const float2 f = Elem<T>::unpack(b[i]);
                            acc[2 * i] = fmaf(wk, f.x, acc[2 * i]); acc[2 * i + 1] = fmaf(wk, f.y, acc[2 * i + 1]);
                        }
                    }
                }
            }
            if (u < u_hi) store_elems<T, V>(out + (size_t)t * H + u * V, acc);
        }
    }
    pdl_launch();
}

// d_rows[r] = w d_out[t] and d_w[t, k] = <d_out[t], rows[r]>: a CTA takes a token, so that the products' sums stay inside it.
template <typename T>
__global__ void __launch_bounds__(256) combine_grad_kernel(const OrderParams o, const T* __restrict__ d_out, const T* __restrict__ rows,
                                                           const float* __restrict__ w, T* __restrict__ d_rows, float* __restrict__ d_w, int H) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float s_dot[2][8][ORDER_MAX_PICKS];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const int units = H / V;
    pdl_wait();
    int buf = 0;
    for (int t = blockIdx.x; t < o.T; t += gridDim.x, buf ^= 1) {
        int rk[ORDER_MAX_PICKS];
        float wk[ORDER_MAX_PICKS], dot[ORDER_MAX_PICKS];
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; ++k) {
            rk[k] = k < o.top_k ? __ldg(o.pair_row + (size_t)t * o.top_k + k) : -1;
            if (rk[k] >= o.num_rows) rk[k] = -1;
            wk[k] = k < o.top_k ? __ldg(w + (size_t)t * o.top_k + k) : 0.f;
            dot[k] = 0.f;
        }
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            float g[V];
            load_elems<T, V>(d_out + (size_t)t * H + u * V, g);
            uint4 v[ORDER_MAX_PICKS];
#pragma unroll
            for (int k = 0; k < ORDER_MAX_PICKS; ++k)
                if (rk[k] >= 0) v[k] = __ldcs(reinterpret_cast<const uint4*>(rows + (size_t)rk[k] * H) + u);
#pragma unroll
            for (int k = 0; k < ORDER_MAX_PICKS; ++k)
                if (rk[k] >= 0) {
                    const uint32_t b[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                    float y[V];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (sizeof(T) == 4) {
                            dot[k] = fmaf(g[i], __uint_as_float(b[i]), dot[k]);
                        } else {
                            const float2 f = Elem<T>::unpack(b[i]);
                            dot[k] = fmaf(g[2 * i], f.x, dot[k]); dot[k] = fmaf(g[2 * i + 1], f.y, dot[k]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) y[i] = wk[k] * g[i];
                    store_elems<T, V>(d_rows + (size_t)rk[k] * H + u * V, y);
                }
        }
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; ++k) {
            for (int off = 16; off; off >>= 1) dot[k] += __shfl_xor_sync(0xFFFFFFFFu, dot[k], off);
            if (lane == 0) s_dot[buf][wid][k] = dot[k];
        }
        __syncthreads();      // (two buffers: a warp is at most one token ahead of the thread that sums)
        if (threadIdx.x < o.top_k) {
            float sum = 0.f;
            for (int i = 0; i < nw; ++i) sum += s_dot[buf][i][threadIdx.x];
            d_w[(size_t)t * o.top_k + threadIdx.x] = sum;
        }
    }
    pdl_launch();
    zero_padding(o, reinterpret_cast<char*>(d_rows), H * (int)sizeof(T) / 32, blockIdx.x * nw + wid, gridDim.x * nw);
}

}  // namespace b200moe
