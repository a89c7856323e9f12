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
// Latency: 56 pairs 2.5 us, 2048 5.8, 32768 6.1, 112856 (over 256 experts) 8.5, against 0.2 us of memory traffic at most.  One CTA for few
// pairs, one meeting less than a kernel more; else two kernels, of which the second has ranked its pairs before it waits for the first.
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ROUNDS = 4;                                 // pairs a thread holds
constexpr int SORT_CHUNK = SORT_ROUNDS * SORT_THREADS;         // pairs of a CTA at a time
constexpr int SORT_ALONE = 2 * SORT_THREADS;                   // most pairs that one CTA sorts alone
static_assert(SORT_ALONE <= SORT_CHUNK, "one CTA holds all of its pairs");

struct SortParams {
    const int32_t* topk_idx;      // [n], n = T K
    int n, num_local, local_offset, align, max_rows;
    int slice;                    // pairs of a CTA, several CTAs only
    int* slices;                  // [CTAs][sort_pitch(num_local)] histogram per slice; several CTAs only
    int32_t *expert_row0, *row_pair, *pair_row;
};

__host__ __device__ constexpr int sort_pitch(int num_local) { return (num_local + 3) & ~3; }

// Pairs of a thread in the chunk that starts at `begin`: as few as reach its end
__device__ __forceinline__ int sort_rounds(int begin, int end) { return min((end - begin + SORT_THREADS - 1) / SORT_THREADS, SORT_ROUNDS); }

// Ranks of up to SORT_CHUNK pairs from `begin` on: a warp takes 32 consecutive ones for each round and counts per expert in its
// row of wcnt; a pair's rank among the warp's pairs of its expert is the count before its round + the lanes before it (match, popcount).
__device__ __forceinline__ void sort_rank(const SortParams& p, int begin, int end, uint16_t (*wcnt)[ORDER_MAX_LOCAL + 2], int* le, int* rank) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rounds = sort_rounds(begin, end), first = begin + warp * (32 * rounds);
#pragma unroll
    for (int m = 0; m < SORT_ROUNDS; ++m) {
        const int i = first + m * 32 + lane;
        const bool on = m < rounds && i < end;
        const int e = on ? __ldcg(p.topk_idx + i) : 0;
        le[m] = on && e >= p.local_offset && (unsigned)e - (unsigned)p.local_offset < (unsigned)p.num_local ? e - p.local_offset : -1;
        rank[m] = 0;
    }
    for (int e = lane; e < p.num_local; e += 32) wcnt[warp][e] = 0;
    __syncwarp();
#pragma unroll
    for (int m = 0; m < SORT_ROUNDS; ++m) {
        if (m >= rounds || first + m * 32 >= end) break;          // the same for the whole warp
        const unsigned same = __match_any_sync(0xFFFFFFFFu, le[m] >= 0 ? le[m] : -1 - lane);
        const int before = le[m] >= 0 ? wcnt[warp][le[m]] : 0, in = __popc(same & ((1u << lane) - 1u));
        rank[m] = before + in;
        __syncwarp();
        if (le[m] >= 0 && in == 0) wcnt[warp][le[m]] = (uint16_t)(before + __popc(same));
        __syncwarp();
    }
}

// Exclusive prefix over the warps of an expert's counts (thread e: expert e); returns the expert's number of pairs
__device__ __forceinline__ int sort_over_warps(uint16_t (*wcnt)[ORDER_MAX_LOCAL + 2], int e) {
    int r = 0;
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) { const int v = wcnt[w][e]; wcnt[w][e] = (uint16_t)r; r += v; }
    return r;
}

// Exclusive prefix of the padded counts (thread e < ORDER_MAX_LOCAL: expert e's, 0 behind the last), for all threads of the CTA, which meet here
__device__ __forceinline__ int sort_rows_before(int count, int align, int* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int padded = (count + align - 1) & -align;
    int upto = padded;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, off);
        if (lane >= off) upto += v;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int r = upto - padded;
#pragma unroll
    for (int w = 0; w < ORDER_MAX_LOCAL / 32; ++w) r += w < warp ? s_warp[w] : 0;
    return r;
}

// Rows of the pairs that sort_rank saw: next[e] = row of the expert's first pair among them
__device__ __forceinline__ void sort_store(const SortParams& p, int begin, int end, const int* next, uint16_t (*wcnt)[ORDER_MAX_LOCAL + 2], const int* le,
                                           const int* rank) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rounds = sort_rounds(begin, end);
#pragma unroll
    for (int m = 0; m < SORT_ROUNDS; ++m) {
        const int i = begin + (warp * rounds + m) * 32 + lane;
        if (m < rounds && i < end) {
            int r = le[m] >= 0 ? next[le[m]] + wcnt[warp][le[m]] + rank[m] : -1;
            if (r >= p.max_rows) r = -1;
            p.pair_row[i] = r;
            if (r >= 0) p.row_pair[r] = i;
        }
    }
}

// One CTA for up to SORT_ALONE pairs
__global__ void __launch_bounds__(SORT_THREADS) sort_one_kernel(const SortParams p) {
    __shared__ int s_next[ORDER_MAX_LOCAL], s_warp[SORT_WARPS];
    __shared__ uint16_t s_wcnt[SORT_WARPS][ORDER_MAX_LOCAL + 2];
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_launch();
    int le[SORT_ROUNDS], rank[SORT_ROUNDS];
    sort_rank(p, 0, p.n, s_wcnt, le, rank);
    for (int r = tid; r < p.max_rows; r += SORT_THREADS) p.row_pair[r] = -1;
    __syncthreads();
    const int count = tid < p.num_local ? sort_over_warps(s_wcnt, tid) : 0;
    const int r0 = sort_rows_before(count, p.align, s_warp);
    if (tid < p.num_local) s_next[tid] = r0;
    if (tid <= p.num_local) p.expert_row0[tid] = min(r0, p.max_rows);
    __syncthreads();
    sort_store(p, 0, p.n, s_next, s_wcnt, le, rank);
}

// Several CTAs, first kernel: the slice's histogram; row_pair is cleared for the second one.
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortParams p) {
    __shared__ int s_count[ORDER_MAX_LOCAL];
    const int tid = threadIdx.x;
    const int pitch = sort_pitch(p.num_local);
    if (tid < pitch) s_count[tid] = 0;
    pdl_wait();
    pdl_launch();
    __syncthreads();
    const long long begin = (long long)blockIdx.x * p.slice;
    const int end = (int)min((long long)p.n, begin + p.slice);
    for (long long i = begin + tid; i < end; i += SORT_THREADS) {
        const int e = __ldg(p.topk_idx + i);
        if (e >= p.local_offset && (unsigned)e - (unsigned)p.local_offset < (unsigned)p.num_local) atomicAdd(s_count + (e - p.local_offset), 1);
    }
    for (long long r = blockIdx.x * (long long)SORT_THREADS + tid; r < p.max_rows; r += gridDim.x * (long long)SORT_THREADS) p.row_pair[r] = -1;
    __syncthreads();
    if (tid < pitch) p.slices[(size_t)blockIdx.x * pitch + tid] = s_count[tid];
}

// Second kernel: every CTA sums the histograms (all of them: the first rows; those before its own: where its pairs start
// inside a segment) and places its slice.  No CTA waits for another.
__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(const SortParams p) {
    __shared__ int s_count[ORDER_MAX_LOCAL], s_next[ORDER_MAX_LOCAL], s_warp[SORT_WARPS];
    __shared__ uint16_t s_wcnt[SORT_WARPS][ORDER_MAX_LOCAL + 2];
    const int tid = threadIdx.x, El = p.num_local, c = blockIdx.x;
    if (tid < ORDER_MAX_LOCAL) { s_count[tid] = 0; s_next[tid] = 0; }
    const int begin = (int)((long long)c * p.slice), end = (int)min((long long)p.n, (long long)begin + p.slice);
    int le[SORT_ROUNDS], rank[SORT_ROUNDS];
    // The ids were there before any CTA of the first kernel let this one start; they are read past L1.
    sort_rank(p, begin, end, s_wcnt, le, rank);
    __syncthreads();
    pdl_wait();
    pdl_launch();
    // four experts per load, eight rows of the table in flight (111 slices of 256 experts: 8 us with one expert per load)
    const int quads = sort_pitch(El) >> 2;
    int width = 8;                                    // threads of one row of the table
    while (width < quads) width <<= 1;
    const int e4 = tid & (width - 1);
    if (e4 < quads) {
        int total[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
#pragma unroll 8
        for (int s = tid / width; s < (int)gridDim.x; s += SORT_THREADS / width) {
            const int4 v = __ldcg(reinterpret_cast<const int4*>(p.slices) + (size_t)s * quads + e4);
            const int first = s < c;
            total[0] += v.x; total[1] += v.y; total[2] += v.z; total[3] += v.w;
            before[0] += first * v.x; before[1] += first * v.y; before[2] += first * v.z; before[3] += first * v.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (total[i]) atomicAdd(s_count + 4 * e4 + i, total[i]);
            if (before[i]) atomicAdd(s_next + 4 * e4 + i, before[i]);
        }
    }
    int here = tid < El ? sort_over_warps(s_wcnt, tid) : 0;
    __syncthreads();
    const int r0 = sort_rows_before(tid < El ? s_count[tid] : 0, p.align, s_warp);
    if (tid < El) s_next[tid] += r0;
    if (c == 0 && tid <= El) p.expert_row0[tid] = min(r0, p.max_rows);
    __syncthreads();
    sort_store(p, begin, end, s_next, s_wcnt, le, rank);
    for (int at = begin + SORT_CHUNK; at < end; at += SORT_CHUNK) {      // (a slice is no longer than 2^30, so `at` stays below 2^31)
        __syncthreads();
        if (tid < El) s_next[tid] += here;
        sort_rank(p, at, end, s_wcnt, le, rank);
        __syncthreads();
        here = tid < El ? sort_over_warps(s_wcnt, tid) : 0;
        __syncthreads();
        sort_store(p, at, end, s_next, s_wcnt, le, rank);
    }
}

// ---------------------------------------------------------------- rows into expert order
struct OrderParams {
    const int32_t* expert_row0;   // [num_local + 1]
    const int32_t* row_pair;      // [num_rows]
    const int32_t* pair_row;      // [T, top_k]
    int T, top_k, num_local, num_rows;
};

// Byte work, bound by HBM: at 7168 bf16 columns and 8 rows per token, 256 experts, permute 8192 tokens 168 us (6.5 TB/s of what it cannot do
// without, 99 % of the copy rate measured on the same kind of card), restore 4096: 83 us (97 %), combine 4096: 79 us (102 %), its gradient 164 us
// (96 %).  Every row crosses memory once (counters: bytes read and written within 1 % of the operands'), nothing is staged in shared memory:
// the rows of a token are independent streams, and loads in flight are what fills the bus.  A warp per token (the first form) left lanes and steps
// of a row empty and paid the look-up of its rows once per token: 183, 105, 91 and 166 us.
//
// The row kernels below deal 32-byte units (16 columns of 16 bits, 8 of 32) of all tokens' rows out to consecutive threads, so that
// no width leaves lanes idle: unit g belongs to token g / units.
struct Unit { int token, unit; };
__device__ __forceinline__ Unit unit_of(unsigned long long g, unsigned units) {
    const unsigned t = g >> 32 ? (unsigned)(g / units) : (unsigned)g / units;
    return {(int)t, (int)(g - (unsigned long long)t * units)};
}

// Rows of token t, -1 where a pick has none.  (Four picks per load where the table allows it.)
__device__ __forceinline__ void token_rows(const OrderParams& o, int t, int* r) {
    const int32_t* src = o.pair_row + (size_t)t * o.top_k;
    if (o.top_k % 4 == 0 && (reinterpret_cast<uintptr_t>(o.pair_row) & 15) == 0) {
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; k += 4) {
            const int4 q = k < o.top_k ? __ldg(reinterpret_cast<const int4*>(src + k)) : make_int4(-1, -1, -1, -1);
            r[k] = q.x; r[k + 1] = q.y; r[k + 2] = q.z; r[k + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; ++k) r[k] = k < o.top_k ? __ldg(src + k) : -1;
    }
#pragma unroll
    for (int k = 0; k < ORDER_MAX_PICKS; ++k)
        if (r[k] >= o.num_rows) r[k] = -1;
}

// Zeros into the padding rows of the segments: rows in use whose pair is none of the T K (-1, or an id of another call's tables).  Every warp owns a
// block of up to 32 consecutive rows (several where there are more rows than that).  Which rows of the first block are padding is looked up
// early (begin) and acted on behind the kernel's own work, so that the look-up's latency hides.
// APART: the warps of a CTA own blocks that are a grid apart, so that one SM does not get the padding of a whole segment: permute with CTAs of 128 threads one token
// 2.9 -> 2.3 us, 512 tokens 19.1 -> 18.2.  (The gradient of the combine stores all of its rows by tokens and is better off with blocks side by side: 2500
// tokens of 128 columns 4.9 us, 6.0 with blocks apart.)
template <bool APART>
struct Padding {
    int used;
    bool empty;                                        // this lane's row of the block
    static __device__ __forceinline__ int warp() {
        if constexpr (APART) return (int)((threadIdx.x >> 5) * gridDim.x + blockIdx.x);
        return (int)((blockIdx.x * (unsigned long long)blockDim.x + threadIdx.x) >> 5);
    }
    static __device__ __forceinline__ int warps() { return (int)((gridDim.x * (unsigned long long)blockDim.x) >> 5); }
    static __device__ __forceinline__ int per(const OrderParams& o) { return min(32, (o.num_rows - 1) / warps() + 1); }
    __device__ __forceinline__ void look(const OrderParams& o, long long r0, int n) {
        const int lane = threadIdx.x & 31;
        empty = lane < n && r0 + lane < used && (unsigned)__ldg(o.row_pair + r0 + lane) >= (unsigned)(o.T * o.top_k);
    }
    __device__ __forceinline__ void begin(const OrderParams& o) {
        used = min(__ldg(o.expert_row0 + o.num_local), o.num_rows);
        const int n = per(o);
        look(o, (long long)warp() * n, n);
    }
    __device__ __forceinline__ void fill(const OrderParams& o, char* rows, int units) {
        const int lane = threadIdx.x & 31, n = per(o);
        for (long long r0 = (long long)warp() * n;;) {
            for (unsigned left = __ballot_sync(0xFFFFFFFFu, empty); left; left &= left - 1) {
                char* dst = rows + (size_t)(r0 + __ffs(left) - 1) * units * 32;
                for (int u = lane; u < units; u += 32) st_global_v8(dst + (size_t)u * 32, 0, 0, 0, 0, 0, 0, 0, 0);
            }
            r0 += (long long)warps() * n;
            if (r0 >= used) break;
            look(o, r0, n);
        }
    }
};

// rows[r] = x[t] for the token's rows: a unit is read once and stored up to top_k times.  The CTA's size is the host's choice (unit_block).
constexpr int PERMUTE_THREADS = 256;         // most threads of a CTA
__global__ void __launch_bounds__(PERMUTE_THREADS) permute_rows_kernel(const OrderParams o, const char* __restrict__ x, char* __restrict__ rows, int units) {
    pdl_wait();
    Padding<true> pad;
    pad.begin(o);
    const unsigned long long total = (unsigned long long)o.T * units, step = (unsigned long long)gridDim.x * blockDim.x;
    for (unsigned long long g = blockIdx.x * (unsigned long long)blockDim.x + threadIdx.x; g < total; g += step) {
        const Unit at = unit_of(g, units);
        uint32_t v[8];
        ld_global_v8(x + g * 32, v);
        int r[ORDER_MAX_PICKS];
        token_rows(o, at.token, r);
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; ++k)
            if (r[k] >= 0) st_global_v8(rows + ((size_t)r[k] * units + at.unit) * 32, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
    }
    pdl_launch();
    pad.fill(o, rows, units);
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

// rows[r] = q[t] * scale, like permute_rows_kernel with units of 16 columns.  Without an order (pair_row null) row t is token t.
template <typename T>
__global__ void __launch_bounds__(PERMUTE_THREADS) restore_rows_kernel(const OrderParams o, const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                           T* __restrict__ rows, int H) {
    pdl_wait();
    const bool ordered = o.pair_row != nullptr;
    const int units = H >> 4;
    Padding<true> pad;
    if (ordered) pad.begin(o);
    const unsigned long long total = (unsigned long long)o.T * units, step = (unsigned long long)gridDim.x * blockDim.x;
    for (unsigned long long g = blockIdx.x * (unsigned long long)blockDim.x + threadIdx.x; g < total; g += step) {
        const Unit at = unit_of(g, units);
        const uint4 b = __ldg(reinterpret_cast<const uint4*>(q) + g);
        const float s = __ldg(scale + (size_t)(at.unit >> 3) * o.T + at.token);
        float v[16];
        if (!ordered) {
            restore16(b, s, v);
            store_elems<T, 16>(rows + g * 16, v);
            continue;
        }
        int r[ORDER_MAX_PICKS];
        token_rows(o, at.token, r);
        restore16(b, s, v);
#pragma unroll
        for (int k = 0; k < ORDER_MAX_PICKS; ++k)
            if (r[k] >= 0) store_elems<T, 16>(rows + (size_t)r[k] * H + at.unit * 16, v);
    }
    pdl_launch();
    if (ordered) pad.fill(o, reinterpret_cast<char*>(rows), H * (int)sizeof(T) / 32);
}

// ---------------------------------------------------------------- rows back to their tokens
// out[t] = sum_k w[t, k] rows[r(t, k)], w null: ones.  A thread takes 32-byte units, one after the other: while the rows of one are on their
// way it looks up the rows of the next, so that the chain of dependent loads is paid once; up to eight rows' loads are in flight, which four
// CTAs of 128 threads per SM leave registers for (two of 256: 1 token 2.1 us against 1.9, 1500 tokens 6.5 against 6.2).  4096 tokens of 7168 columns: all eight rows here 79 us, half of them 47, an eighth 30 (a
// floor of 18: a thread then has one load in flight, but three or four CTAs with fewer loads each took 28 to 29 and cost the full case 8 us, and a
// warp per token with four units in flight 33).
constexpr int COMBINE_THREADS = 128, COMBINE_CTAS = 4;         // CTAs of an SM
template <typename T>
__global__ void __launch_bounds__(COMBINE_THREADS, COMBINE_CTAS) combine_rows_kernel(const OrderParams o, const T* __restrict__ rows, const float* __restrict__ w,
                                                              T* __restrict__ out, int H) {
    constexpr int V = 32 / sizeof(T), K = ORDER_MAX_PICKS;
    pdl_wait();
    const int units = H / V;
    const unsigned long long total = (unsigned long long)o.T * units, step = (unsigned long long)gridDim.x * blockDim.x;
    unsigned long long g = blockIdx.x * (unsigned long long)blockDim.x + threadIdx.x;
    if (g < total) {
        Unit at = unit_of(g, units);
        int r[K];
        token_rows(o, at.token, r);
        while (true) {
            const unsigned long long next = g + step;
            Unit at2 = {0, 0};
            int r2[K];
            uint32_t v[K][8];
            float wk[K], acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (r[k] >= 0) {
                    ld_global_v8(rows + (size_t)r[k] * H + at.unit * V, v[k]);
                    wk[k] = w ? __ldg(w + (size_t)at.token * o.top_k + k) : 1.f;
                }
            if (next < total) {
                at2 = unit_of(next, units);
                token_rows(o, at2.token, r2);
            }
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (r[k] >= 0)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (sizeof(T) == 4) {
                            acc[i] = fmaf(wk[k], __uint_as_float(v[k][i]), acc[i]);
                        } else {
                            const float2 f = Elem<T>::unpack(v[k][i]);
                            acc[2 * i] = fmaf(wk[k], f.x, acc[2 * i]); acc[2 * i + 1] = fmaf(wk[k], f.y, acc[2 * i + 1]);
                        }
                    }
            store_elems<T, V>(out + g * V, acc);
            if (next >= total) break;
            g = next; at = at2;
#pragma unroll
            for (int k = 0; k < K; ++k) r[k] = r2[k];
        }
    }
    pdl_launch();
}

// Sums of eight values over the 32 lanes in nine shuffles instead of forty: three steps halve what a lane carries, two more add.  Lane l
// returns the sum of value l >> 2.
__device__ __forceinline__ float warp_sums8(const float* v, int lane) {
    float a[4], b[2], c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float keep = lane & 16 ? v[i + 4] : v[i], give = lane & 16 ? v[i] : v[i + 4];
        a[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float keep = lane & 8 ? a[i + 2] : a[i], give = lane & 8 ? a[i] : a[i + 2];
        b[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 8);
    }
    {
        const float keep = lane & 4 ? b[1] : b[0], give = lane & 4 ? b[0] : b[1];
        c = keep + __shfl_xor_sync(0xFFFFFFFFu, give, 4);
    }
    c += __shfl_xor_sync(0xFFFFFFFFu, c, 2);
    return c + __shfl_xor_sync(0xFFFFFFFFu, c, 1);
}

// 16 bytes of a row as fp32 values
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& q, float* v) {
    const uint32_t b[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(b[i]);
        } else {
            const float2 f = Elem<T>::unpack(b[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}

// One unit of one row: its part of the product's sum, and w times the gradient stored
template <typename T>
__device__ __forceinline__ float grad_unit(const float* g, const uint4& row, float w, T* dst, float dot) {
    constexpr int V = 16 / sizeof(T);
    float y[V];
    unpack16<T>(row, y);
#pragma unroll
    for (int i = 0; i < V; ++i) { dot = fmaf(g[i], y[i], dot); y[i] = w * g[i]; }
    store_elems<T, V>(dst, y);
    return dot;
}

// d_rows[r] = w d_out[t] and d_w[t, k] = <d_out[t], rows[r]>, two ways.
// By tokens: a group of threads (whole warps) takes a token with all of its rows, so that d_out is read once and eight rows' loads are in
// flight.  By rows: a group takes a row, with FLIGHT units of it in flight per thread, whichever token it belongs to; d_out comes from L2
// as often as it has rows.
constexpr int GRAD_FLIGHT = 4, GRAD_THREADS = 128, GRAD_WARPS = GRAD_THREADS / 32;
template <typename T>
__device__ __forceinline__ void combine_grad_by_rows(const OrderParams& o, const T* __restrict__ d_out, const T* __restrict__ rows, const float* __restrict__ w,
                                                     T* __restrict__ d_rows, float* __restrict__ d_w, int H, int gsh, int used, float (*s_dot)[GRAD_WARPS][ORDER_MAX_PICKS]) {
    constexpr int V = 16 / sizeof(T), FLIGHT = GRAD_FLIGHT;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int groups = GRAD_THREADS >> gsh, stride = 1 << gsh, in = threadIdx.x & (stride - 1);
    const int units = H / V, pairs = o.T * o.top_k;
    for (long long i = blockIdx.x * (long long)GRAD_THREADS + threadIdx.x; i < pairs; i += gridDim.x * (long long)GRAD_THREADS) {
        const int r = __ldg(o.pair_row + i);
        if (r < 0 || r >= o.num_rows) d_w[i] = 0.f;
    }
    int buf = 0;
    const long long step = (long long)gridDim.x * groups, r_first = (long long)blockIdx.x * groups + (threadIdx.x >> gsh);
    int next = r_first < used ? __ldg(o.row_pair + r_first) : -1;          // the next row's pair, looked up one turn ahead
    for (long long r0 = (long long)blockIdx.x * groups; r0 < used; r0 += step, buf ^= 1) {
        const long long r = r0 + (threadIdx.x >> gsh);
        const int pair = next < pairs ? next : -1;                            // (negative: none)
        next = r + step < used ? __ldg(o.row_pair + r + step) : -1;
        float dot = 0.f;
        if (r < used) {
            T* dst = d_rows + (size_t)r * H;
            if (pair < 0) {
                for (int u = in; u < units / 2; u += stride) st_global_v8(reinterpret_cast<char*>(dst) + (size_t)u * 32, 0, 0, 0, 0, 0, 0, 0, 0);
            } else {
                const float wk = __ldg(w + pair);
                const uint4 *src = reinterpret_cast<const uint4*>(d_out + (size_t)(pair / o.top_k) * H),
                            *row = reinterpret_cast<const uint4*>(rows + (size_t)r * H);
                for (int u0 = in; u0 < units; u0 += FLIGHT * stride) {
                    uint4 d[FLIGHT], v[FLIGHT];
#pragma unroll
                    for (int q = 0; q < FLIGHT; ++q)
                        if (u0 + q * stride < units) { d[q] = __ldg(src + u0 + q * stride); v[q] = __ldcs(row + u0 + q * stride); }
#pragma unroll
                    for (int q = 0; q < FLIGHT; ++q)
                        if (u0 + q * stride < units) {
                            float g[V];
                            unpack16<T>(d[q], g);
                            dot = grad_unit<T>(g, v[q], wk, dst + (u0 + q * stride) * V, dot);
                        }
                }
            }
        }
        for (int off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, off);
        if (gsh > 5) {
            if (lane == 0) s_dot[buf][wid][0] = dot;
            __syncthreads();
            if (in == 0) {
                dot = 0.f;
                for (int i = 0; i < stride >> 5; ++i) dot += s_dot[buf][wid + i][0];
            }
        }
        if (in == 0 && pair >= 0) d_w[pair] = dot;
    }
}

template <typename T>
__device__ __forceinline__ void combine_grad_by_tokens(const OrderParams& o, const T* __restrict__ d_out, const T* __restrict__ rows, const float* __restrict__ w,
                                                       T* __restrict__ d_rows, float* __restrict__ d_w, int H, int gsh, float (*s_dot)[GRAD_WARPS][ORDER_MAX_PICKS]) {
    constexpr int V = 16 / sizeof(T), K = ORDER_MAX_PICKS;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int group = threadIdx.x >> gsh, groups = GRAD_THREADS >> gsh, stride = 1 << gsh, in = threadIdx.x & (stride - 1);
    const int units = H / V;
    int buf = 0;
    for (long long t0 = (long long)blockIdx.x * groups; t0 < o.T; t0 += (long long)gridDim.x * groups, buf ^= 1) {
        const long long t = t0 + group;
        int r[K];
        float wk[K], dot[K];
#pragma unroll
        for (int k = 0; k < K; ++k) { r[k] = -1; dot[k] = 0.f; }
        if (t < o.T) {
            token_rows(o, (int)t, r);
#pragma unroll
            for (int k = 0; k < K; ++k) wk[k] = k < o.top_k ? __ldg(w + (size_t)t * o.top_k + k) : 0.f;
            for (int u = in; u < units; u += stride) {
                float g[V];
                load_elems<T, V>(d_out + (size_t)t * H + u * V, g);
                uint4 v[K];
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (r[k] >= 0) v[k] = __ldcs(reinterpret_cast<const uint4*>(rows + (size_t)r[k] * H) + u);
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (r[k] >= 0) dot[k] = grad_unit<T>(g, v[k], wk[k], d_rows + (size_t)r[k] * H + u * V, dot[k]);
            }
        }
        const float sum = warp_sums8(dot, lane);          // of row lane >> 2
        if (gsh == 5) {
            if (t < o.T && (lane & 3) == 0 && lane >> 2 < o.top_k) d_w[(size_t)t * o.top_k + (lane >> 2)] = sum;
        } else {
            if ((lane & 3) == 0) s_dot[buf][wid][lane >> 2] = sum;
            __syncthreads();
            if (t < o.T && in < o.top_k) {
                float total = 0.f;
                for (int i = 0; i < stride >> 5; ++i) total += s_dot[buf][(group << (gsh - 5)) + i][in];
                d_w[(size_t)t * o.top_k + in] = total;
            }
        }
    }
}

// By rows for few tokens, and where few of the picks have a row here (an expert-parallel rank's share).  By tokens / by rows, us, 8 picks of 256 experts, all
// here: 7168 columns one token 8.6 / 2.6, 64: 17.1 / 17.1, 128: 19.5 / 19.9, 256: 22.6 / 22.7, 512: 31.4 / 32.8, 1024: 49.8 / 51.7, 4096: 165 / 195; 2048 columns 64:
// 7.3 / 5.3, 256: 8.5 / 6.7, 512: 12.0 / 11.5, 1024: 16.3 / 18.2; 256 columns 256: 3.1 / 2.8, 512: 3.4 / 3.6, 1024: 3.9 / 5.4.
// 4096 tokens with one / two / three / four rows each: 7168 columns 57 / 29, 69 / 50, 81 / 73, 95 / 95; 2048 columns 22 / 9, 26 / 16, 29 / 22, 33 / 28; 256 columns
// 4.8 / 3.5, 5.2 / 5.3, 5.4 / 7.0, 5.8 / 9.4: a line (rows in use, padding counted) between what wide and narrow rows ask for.
// Groups of 2^row_sh or 2^token_sh threads; with 256 threads per CTA, two tokens that wait for each other in every turn, 512 tokens took 33.8 us (31.1
// with 128), 4096: 165.9 (164.4), 64, by rows, 17.6 (17.2).
// In both ways all threads of a CTA make the same number of turns, as they meet in each; the sums' two buffers let a warp be one turn
// ahead of the thread that reads them.
constexpr int GRAD_FEW_TOKENS = 256, GRAD_FEW_ROWS = 3;
template <typename T>
__global__ void __launch_bounds__(GRAD_THREADS, 4) combine_grad_kernel(const OrderParams o, const T* __restrict__ d_out, const T* __restrict__ rows,
                                                              const float* __restrict__ w, T* __restrict__ d_rows, float* __restrict__ d_w, int H,
                                                              int token_sh, int row_sh) {
    __shared__ float s_dot[2][GRAD_WARPS][ORDER_MAX_PICKS];
    pdl_wait();
    const int used = min(__ldg(o.expert_row0 + o.num_local), o.num_rows);
    if (o.T <= GRAD_FEW_TOKENS || used <= (long long)GRAD_FEW_ROWS * o.T) {
        combine_grad_by_rows(o, d_out, rows, w, d_rows, d_w, H, row_sh, used, s_dot);
        pdl_launch();
    } else {
        Padding<false> pad;
        pad.begin(o);
        combine_grad_by_tokens(o, d_out, rows, w, d_rows, d_w, H, token_sh, s_dot);
        pdl_launch();
        pad.fill(o, reinterpret_cast<char*>(d_rows), H * (int)sizeof(T) / 32);
    }
}

}  // namespace b200moe
