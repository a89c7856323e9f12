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
// restored as an infinity (off by less than 2^-4, like any other code).  A group that holds an infinity or a NaN gets the scale NaN: its values
// are gone, and the gradients made from it say so instead of being finite.
// Byte work: 2048 columns of bf16, 34645 rows in use, save 91 us, backward with the activation 110 us in a row of such calls: 96 and 100 % of
// the measured copy rate over the bytes that have to move; 8000 rows 24 and 28 us (83 and 89 %), 20000 rows of 256 columns 10 and 11 us.  The
// save kernel issues in 64 % of its cycles (counters), so the arithmetic is kept short: products with powers of two instead of divisions, the
// fast exponential for 16-bit rows.
#pragma once
#include "order.cuh"

namespace b200moe {

constexpr int SWIGLU_THREADS = 256, SWIGLU_LANES = 8;        // lanes of a group of 128 columns, 16 each
constexpr int SWIGLU_TURN = SWIGLU_THREADS / SWIGLU_LANES;   // pairs of groups a CTA takes at a time
constexpr int SWIGLU_SCALES = 512;                           // most pairs of groups of a CTA

// 1 / (1 + exp(-g)).  For 16-bit rows with the fast exponential and quotient: a few units of 2^-22, and where the quotient flushes to zero
// (1 + exp(-g) above 2^126) the product is below every value of those types.  fp32 rows take the accurate ones.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    if constexpr (sizeof(T) == 4) return __fdiv_rn(1.0f, 1.0f + expf(-g));
    return __fdividef(1.0f, 1.0f + __expf(-g));
}

// Exponent e of a group's scale 2^e from its largest magnitude (finite, not negative): amax = m 2^x with m in [1, 2), 448 = 1.75 2^8,
// so amax / 448 <= 2^(x - 8) exactly if m <= 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    return max((int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u), -126);
}

// Largest magnitude of 16 values and over the eight lanes of a group; NaN where there is one
__device__ __forceinline__ float group_amax(const float* v) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[i])));
#pragma unroll
    for (int o = 4; o; o >>= 1) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(__shfl_xor_sync(0xFFFFFFFFu, m, o)));
    return m;
}

// Codes of 16 values of a group, and its scale
__device__ __forceinline__ uint4 encode16(const float* v, float amax, float& scale) {
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
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)f32x2_to_e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | ((uint32_t)f32x2_to_e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
    if (top)                     // 0x77 is 240
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __vminu4(w[i] & 0x7F7F7F7Fu, 0x77777777u) | (w[i] & 0x80808080u);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// CTA (x, y): rows [x rpc, ...), pairs of groups [y gpc, ...), rpc = 2^rsh, rpc gpc <= SWIGLU_SCALES.  Eight lanes own column
// group j of up and of gate, 32 bytes (16-bit types) of each per lane; scales wait in shared memory until a group's run of rows
// leaves as one store.
template <typename T>
__global__ void __launch_bounds__(SWIGLU_THREADS) swiglu_save_kernel(const T* __restrict__ x, const int32_t* __restrict__ used, int rows, int I, int rsh,
                                                                     int gpc, T* __restrict__ act, uint8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ float s_scale[2][SWIGLU_SCALES];      // [up, gate][group][row]
    const int groups = I >> 7, sub = threadIdx.x & 7;
    const int r0 = blockIdx.x << rsh, j0 = blockIdx.y * gpc;
    pdl_wait();
    const int live = used ? min(__ldg(used), rows) : rows;
    const int nr = min(1 << rsh, live - r0), nj = min(gpc, groups - j0);
    if (nr <= 0) return;
    const int total = nr * nj;
    // the trip count is the same for all lanes (the shuffles name the warp)
    for (int i0 = 0; i0 < total; i0 += SWIGLU_TURN) {
        const int i = i0 + (threadIdx.x >> 3);
        const int r = i / nj, j = i - r * nj;
        const bool on = i < total;
        const size_t at = (size_t)(r0 + r) * 2 * I + (size_t)(j0 + j) * 128 + sub * 16;
        float up[16], gate[16];
        if (on) {
            load_elems<T, 16>(x + at, up);
            load_elems<T, 16>(x + at + I, gate);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) up[k] = gate[k] = 0.f;
        }
        const float mu = group_amax(up), mg = group_amax(gate);
        if (!on) continue;
        float su, sg;
        *reinterpret_cast<uint4*>(q + at) = encode16(up, mu, su);
        *reinterpret_cast<uint4*>(q + at + I) = encode16(gate, mg, sg);
#pragma unroll
        for (int k = 0; k < 16; ++k) up[k] *= gate[k] * sigmoid<T>(gate[k]);
        store_elems<T, 16>(act + (size_t)(r0 + r) * I + (size_t)(j0 + j) * 128 + sub * 16, up);
        if (sub == 0) { s_scale[0][(j << rsh) + r] = su; s_scale[1][(j << rsh) + r] = sg; }
    }
    __syncthreads();
    pdl_launch();
    for (int i = threadIdx.x; i < nj << rsh; i += SWIGLU_THREADS) {
        const int j = i >> rsh, r = i - (j << rsh);
        if (r < nr) {
            scale[(size_t)(j0 + j) * rows + r0 + r] = s_scale[0][i];
            scale[(size_t)(groups + j0 + j) * rows + r0 + r] = s_scale[1][i];
        }
    }
}

template <typename T, bool ACT>
__global__ void __launch_bounds__(SWIGLU_THREADS) swiglu_grad_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scale, const T* __restrict__ d_act,
                                                                     const int32_t* __restrict__ used, int rows, int I, int rsh, int gpc,
                                                                     T* __restrict__ d_x, T* __restrict__ act) {
    const int groups = I >> 7, sub = threadIdx.x & 7;
    const int r0 = blockIdx.x << rsh, j0 = blockIdx.y * gpc;
    pdl_wait();
    const int live = used ? min(__ldg(used), rows) : rows;
    const int nr = min(1 << rsh, live - r0), nj = min(gpc, groups - j0);
    const int total = nr > 0 ? nr * nj : 0;
    for (int i = threadIdx.x >> 3; i < total; i += SWIGLU_TURN) {
        const int r = i / nj, j = i - r * nj;
        const size_t at = (size_t)(r0 + r) * 2 * I + (size_t)(j0 + j) * 128 + sub * 16;
        const size_t at1 = (size_t)(r0 + r) * I + (size_t)(j0 + j) * 128 + sub * 16;
        float up[16], gate[16], d[16];
        const uint4 qu = __ldg(reinterpret_cast<const uint4*>(q + at)), qg = __ldg(reinterpret_cast<const uint4*>(q + at + I));
        const float su = __ldg(scale + (size_t)(j0 + j) * rows + r0 + r), sg = __ldg(scale + (size_t)(groups + j0 + j) * rows + r0 + r);
        load_elems<T, 16>(d_act + at1, d);
        restore16(qu, su, up);
        restore16(qg, sg, gate);
        float a[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float s = sigmoid<T>(gate[k]), silu = gate[k] * s;
            a[k] = up[k] * silu;
            gate[k] = d[k] * up[k] * (s * fmaf(gate[k], 1.0f - s, 1.0f));
            up[k] = d[k] * silu;
        }
        store_elems<T, 16>(d_x + at, up);
        store_elems<T, 16>(d_x + at + I, gate);
        if constexpr (ACT) store_elems<T, 16>(act + at1, a);
    }
    pdl_launch();
}

}  // namespace b200moe
