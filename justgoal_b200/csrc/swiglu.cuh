// SwiGLU between the two GEMMs, with its inputs kept in 8 bits for the backward pass.
//
// x = [up | gate] of I columns each (the operator's order: act = up * silu(gate)).
//   save      act = up gate sigma(gate) from the unrounded x, and the copy (q, scale) of x: e4m3 codes and one scale per 1x128 group
//   backward  up, gate = q scale; s = sigma(gate): d_up = d gate s, d_gate = d up s (1 + gate (1 - s)), act = up gate s again
//             (GEMM2's weight gradient needs it, and nothing else of the forward pass has to be kept)
//
// scale = the smallest power of two that is not below amax / 448 (at least 2^-126; 1 for a group of zeros): the product
// with 1 / scale is exact, so a code is x / scale rounded once, without a division, and the copy of 16-bit values is restored
// without a rounding.  An e4m3 number has the same relative precision in the upper half of its range as at its end, so the copy loses
// nothing to amax / 448 but one of the 15 binades above its subnormals.  Under the scale 2^120 the codes end at 240, so that no finite value is
// an infinity in fp32 or bf16 when it is restored (off by less than 2^-4, like any other code).  In fp16 one above 63488, whose code stands for 65536, would be; the
// gradient is made from the copy in fp32, where it is finite.  A group that holds an infinity or a NaN gets the scale NaN: its values
// are gone, and the gradients made from it say so instead of being finite.
// Byte work: 2048 columns of bf16, 34645 rows in use, save 88 us, backward with the activation 105 us in a row of such calls: 100 and 104 % of
// the measured copy rate over the bytes that have to move (after a second of load 92 and 108, at the clocks of the power limit); without the activation 84; 8000 rows
// 23 and 26 us (88 and 96 %), 20000 rows of 256 columns 9.0 and 9.8 us.  The arithmetic has to stay out of the way, also at those clocks: products with powers
// of two instead of divisions, two values per instruction, magnitudes compared two 16-bit patterns at a time, flushed approximations for 16-bit rows, no
// division in the walk over a block.  With one value per instruction and the library's exponential and quotient the save kernel issued in 64 % of its
// cycles: 91 and 110 us for short, 97 and 115 after a second of load.
#pragma once
#include "order.cuh"

namespace b200moe {

constexpr int SWIGLU_LANES = 8;                                        // lanes of a group of 128 columns, 16 each
constexpr int SAVE_THREADS = 128, SAVE_TURN = SAVE_THREADS / SWIGLU_LANES;       // pairs of groups a CTA takes at a time
constexpr int GRAD_X_THREADS = 256, GRAD_X_TURN = GRAD_X_THREADS / SWIGLU_LANES;
constexpr int SWIGLU_SCALES = 512;                           // most pairs of groups of a CTA

// Two sigmoids, 1 / (1 + 2^(-g log2 e)).  16-bit rows take the fast exponential and reciprocal, flushed.  The product g log2 e is rounded, which moves the
// exponent by a share of |g|: the sigmoid is off by a share of (4.5 + 1.2 |g|) 2^-23 at most, 2^-18 at g = -20 and 2^-16 at -87, far below the output's
// rounding of 2^-8 or 2^-11.  Where the sigmoid leaves fp32's normal range, for gates below -87, it counts as zero.  fp32 rows take the accurate ones:
// three units of 2^-23 down to -87, fewer bits from there to -88.7, where exp(-g) passes the range, zero below.
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 g) {
    if constexpr (sizeof(T) == 4) return make_float2(__fdiv_rn(1.0f, 1.0f + expf(-g.x)), __fdiv_rn(1.0f, 1.0f + expf(-g.y)));
    const float2 t = __fmul2_rn(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    float2 e, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = __fadd2_rn(e, make_float2(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
    return s;
}

// 16 columns of a row as the words that memory has, and as eight pairs of fp32 values
template <typename T>
struct Cols {
    static constexpr int WORDS = 16 * sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* src) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) ld_global_v8(reinterpret_cast<const uint32_t*>(src) + i, w + i);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return Elem<T>::unpack(w[i]);
    }
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (sizeof(T) == 4) { w[2 * i] = __float_as_uint(v.x); w[2 * i + 1] = __float_as_uint(v.y); }
        else w[i] = Elem<T>::pack(v.x, v.y);
    }
    __device__ __forceinline__ void store(T* dst) const {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8)
            st_global_v8(reinterpret_cast<uint32_t*>(dst) + i, w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5], w[i + 6], w[i + 7]);
    }
};

// Largest magnitudes of two groups of 128 columns, 16 of each per lane of eight.  Magnitudes are compared as bit patterns without the sign, so
// that an infinity lies above all numbers and a NaN above that; two groups of 16-bit values share the words and the shuffles.
template <typename T>
__device__ __forceinline__ void group_amax(const Cols<T>& a, const Cols<T>& b, float& ma, float& mb) {
    constexpr unsigned FULL = 0xFFFFFFFFu;
    if constexpr (sizeof(T) == 4) {
        uint32_t x = 0, y = 0;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            x = __vimax3_u32(x, a.w[i] & 0x7FFFFFFFu, a.w[i + 1] & 0x7FFFFFFFu);
            y = __vimax3_u32(y, b.w[i] & 0x7FFFFFFFu, b.w[i + 1] & 0x7FFFFFFFu);
        }
#pragma unroll
        for (int o = 4; o; o >>= 1) { x = max(x, __shfl_xor_sync(FULL, x, o)); y = max(y, __shfl_xor_sync(FULL, y, o)); }
        ma = __uint_as_float(x); mb = __uint_as_float(y);
    } else {
        uint32_t x = 0, y = 0;                       // two maxima each: of even and of odd columns
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            x = __vimax3_u16x2(x, a.w[i] & 0x7FFF7FFFu, a.w[i + 1] & 0x7FFF7FFFu);
            y = __vimax3_u16x2(y, b.w[i] & 0x7FFF7FFFu, b.w[i + 1] & 0x7FFF7FFFu);
        }
        uint32_t m = __vmaxu2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));      // low half: a's, high half: b's
#pragma unroll
        for (int o = 4; o; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(FULL, m, o));
        const float2 f = Elem<T>::unpack(m);
        ma = f.x; mb = f.y;
    }
}

// Exponent e of a group's scale 2^e from its largest magnitude (finite, not negative): amax = m 2^x with m in [1, 2), 448 = 1.75 2^8,
// so amax / 448 <= 2^(x - 8) exactly if m <= 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    return max((int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u), -126);
}

// Codes of 16 values of a group, and its scale
template <typename T>
__device__ __forceinline__ uint4 encode16(const Cols<T>& c, float amax, float& scale) {
    float inv;
    bool top = false;
    if (!(amax < INFINITY)) {
        scale = inv = __uint_as_float(0x7FC00000u);
    } else {
        const int e = amax > 0.f ? scale_exponent(amax) : 0;
        scale = __uint_as_float((uint32_t)(127 + e) << 23);
        inv = __uint_as_float((uint32_t)(127 - e) << 23);
        top = e == 120;
    }
    const float2 by = make_float2(inv, inv);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __fmul2_rn(c.pair(2 * i), by), b = __fmul2_rn(c.pair(2 * i + 1), by);
        w[i] = (uint32_t)f32x2_to_e4m3x2(a.x, a.y) | ((uint32_t)f32x2_to_e4m3x2(b.x, b.y) << 16);
    }
    if (top)                     // 0x77 is 240
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __vminu4(w[i] & 0x7F7F7F7Fu, 0x77777777u) | (w[i] & 0x80808080u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Pair i of 16 e4m3 values times their scale
__device__ __forceinline__ float2 decode2(const uint4& q, int i, float s) {
    const uint32_t w = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __fmul2_rn(e4m3x2_to_f32x2((uint16_t)(i & 1 ? w >> 16 : w)), make_float2(s, s));
}

// The eight lanes' next (row, group) of a CTA's block, TURN of them further on, without a division per step
template <int TURN>
struct BlockWalk {
    int r, j, dr, dj, nj;
    __device__ __forceinline__ BlockWalk(int nj_) : nj(nj_) {
        const int i = threadIdx.x >> 3;
        r = i / nj; j = i - r * nj;
        dr = TURN / nj; dj = TURN - dr * nj;
    }
    __device__ __forceinline__ void step() {
        r += dr; j += dj;
        if (j >= nj) { j -= nj; ++r; }
    }
};

// CTA (x, y): rows [x rpc, ...), pairs of groups [y gpc, ...), rpc = 2^rsh, rpc gpc <= SWIGLU_SCALES.  Eight lanes own column
// group j of up and of gate, 32 bytes (16-bit types) of each per lane; scales wait in shared memory until a group's run of rows
// leaves as one store.
template <typename T>
__global__ void __launch_bounds__(SAVE_THREADS) swiglu_save_kernel(const T* __restrict__ x, const int32_t* __restrict__ used, int rows, int I, int rsh,
                                                                     int gpc, T* __restrict__ act, uint8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ float s_scale[2][SWIGLU_SCALES];      // [up, gate][group][row]
    const int groups = I >> 7, sub = threadIdx.x & 7;
    const int r0 = blockIdx.x << rsh, j0 = blockIdx.y * gpc;
    pdl_wait();
    const int live = used ? min(__ldg(used), rows) : rows;
    const int nr = min(1 << rsh, live - r0), nj = min(gpc, groups - j0);
    if (nr <= 0) return;
    const int total = nr * nj;
    BlockWalk<SAVE_TURN> at(nj);
    // the trip count is the same for all lanes (the shuffles name the warp)
    for (int i0 = 0; i0 < total; i0 += SAVE_TURN, at.step()) {
        const bool on = at.r < nr;
        const size_t col = (size_t)(j0 + at.j) * 128 + sub * 16, row = r0 + at.r;
        Cols<T> up, gate;
        if (on) {
            up.load(x + row * 2 * I + col);
            gate.load(x + row * 2 * I + I + col);
        } else {
            up.clear(); gate.clear();
        }
        float mu, mg, su, sg;
        group_amax(up, gate, mu, mg);
        if (!on) continue;
        *reinterpret_cast<uint4*>(q + row * 2 * I + col) = encode16(up, mu, su);
        *reinterpret_cast<uint4*>(q + row * 2 * I + I + col) = encode16(gate, mg, sg);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 g = gate.pair(k);
            up.set(k, __fmul2_rn(up.pair(k), __fmul2_rn(g, sigmoid2<T>(g))));
        }
        up.store(act + row * I + col);
        if (sub == 0) { s_scale[0][(at.j << rsh) + at.r] = su; s_scale[1][(at.j << rsh) + at.r] = sg; }
    }
    __syncthreads();
    pdl_launch();
    for (int i = threadIdx.x; i < nj << rsh; i += SAVE_THREADS) {
        const int j = i >> rsh, r = i - (j << rsh);
        if (r < nr) {
            scale[(size_t)(j0 + j) * rows + r0 + r] = s_scale[0][i];
            scale[(size_t)(groups + j0 + j) * rows + r0 + r] = s_scale[1][i];
        }
    }
}

template <typename T, bool ACT>
__global__ void __launch_bounds__(GRAD_X_THREADS) swiglu_grad_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ d_act,
                                                                     const int32_t* __restrict__ used, int rows, int I, int rsh, int gpc,
                                                                     T* __restrict__ d_x, T* __restrict__ act) {
    const int groups = I >> 7, sub = threadIdx.x & 7;
    const int r0 = blockIdx.x << rsh, j0 = blockIdx.y * gpc;
    pdl_wait();
    const int live = used ? min(__ldg(used), rows) : rows;
    const int nr = min(1 << rsh, live - r0), nj = min(gpc, groups - j0);
    const int total = nr > 0 ? nr * nj : 0;
    BlockWalk<GRAD_X_TURN> at(max(nj, 1));
    for (int i = threadIdx.x >> 3; i < total; i += GRAD_X_TURN, at.step()) {
        const size_t col = (size_t)(j0 + at.j) * 128 + sub * 16, row = r0 + at.r;
        const uint4 qu = __ldg(reinterpret_cast<const uint4*>(q + row * 2 * I + col)), qg = __ldg(reinterpret_cast<const uint4*>(q + row * 2 * I + I + col));
        const float su = __ldg(scale + (size_t)(j0 + at.j) * rows + row), sg = __ldg(scale + (size_t)(groups + j0 + at.j) * rows + row);
        Cols<T> d, d_gate, a;
        d.load(d_act + row * I + col);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 u = decode2(qu, k, su), g = decode2(qg, k, sg), dk = d.pair(k), one = make_float2(1.0f, 1.0f);
            const float2 s = sigmoid2<T>(g), silu = __fmul2_rn(g, s);
            const float2 slope = __ffma2_rn(silu, __ffma2_rn(s, make_float2(-1.0f, -1.0f), one), s);      // s (1 + g (1 - s))
            d_gate.set(k, __fmul2_rn(__fmul2_rn(dk, u), slope));
            if constexpr (ACT) a.set(k, __fmul2_rn(u, silu));
            d.set(k, __fmul2_rn(dk, silu));
        }
        d.store(d_x + row * 2 * I + col);
        d_gate.store(d_x + row * 2 * I + I + col);
        if constexpr (ACT) a.store(act + row * I + col);
    }
    pdl_launch();
}

}  // namespace b200moe
