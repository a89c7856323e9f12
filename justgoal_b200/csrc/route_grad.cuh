// Gradient of the routing weights down to the logits.  Eight lanes stand for a token's picks: lane k < top_k holds pick k, its expert, its
// logit and d = the gradient of its weight w (all sums over the token's picks; f = the routed scaling factor).
//
//   sigmoid, normalised (DeepSeek)  w_k = f s_k / S, S = sum_j s_j + 1e-20:  d_logit_k = f s'_k (sum_j (d_k - d_j) s_j + 1e-20 d_k) / S^2
//   softmax, normalised (both)      w = f softmax over the picks:            d_logit_k = f w_k sum_j w_j (d_k - d_j)
//   softmax (default)               w_k = f p_k, p over all experts:         d_logit_i = f p_i (d_i - sum_j p_j d_j), d_i = 0 where not picked
//   sigmoid of one pick             d_logit = f d s';    uniform weights: zeros
//
// Differences of the gradients are taken before they are weighted, and 1 - p of a pick is the sum of the other experts' shares:
// nothing is lost where one pick holds nearly all of the weight.  (Softmax over all experts, then normalised over the picks, adds 1e-20
// to a sum that is at least top_k / 512, which fp32 does not see: the same weights as the softmax over the picks.)  An expert that a
// token picks twice gets the sum of both; ids outside [0, E) carry no weight.
// A token costs E floats written, zeros where nothing was picked, and a chain of dependent loads (pick, logit): a warp takes four
// tokens, clears their rows - one run of memory - while the picks are on their way, and stores the picks' gradients behind that.
// The default form reads the row whole, keeps it in registers and takes one token per warp.  8192 tokens over 256 experts 2.7 us (one token per
// warp, rows cleared first: 5.3), default 6.3; one token 1.6 and 2.0, which is the launch.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace b200moe {

enum : int { RG_DEEPSEEK = 0, RG_RENORM_NAIVE = 1, RG_DEFAULT = 2, RG_RENORMALIZE = 3, RG_LLAMA4 = 4, RG_TOPK = 5, RG_COUNT = 6 };

struct RouteGradParams {
    const float* logits;           // [T, E]
    const __nv_bfloat16* bias;     // [E] or null
    const int32_t* topk_idx;       // [T, top_k]
    const float* d_w;              // [T, top_k]
    float* d_logits;               // [T, E]
    int T, E, top_k;
    float factor;
};

constexpr int ROUTE_GRAD_MAX = 512;      // experts

// Pick k of token t for lane k of eight: id (-1: none), logit, gradient of the weight
struct Pick { int id; float x, d; };
__device__ __forceinline__ Pick load_pick(const RouteGradParams& p, int t, int k, bool with_bias) {
    Pick a = {-1, -INFINITY, 0.f};
    if (t < p.T && k < p.top_k) {
        const int id = __ldg(p.topk_idx + (size_t)t * p.top_k + k);
        if (id >= 0 && id < p.E) {
            a.id = id;
            a.d = __ldg(p.d_w + (size_t)t * p.top_k + k);
            a.x = __ldg(p.logits + (size_t)t * p.E + id);
            if (with_bias && p.bias) a.x = __fadd_rn(a.x, __bfloat162float(p.bias[id]));
        }
    }
    return a;
}

// Sum of v over the lanes of the eight that picked the same expert, and whether this lane is the first of them (it stores the sum)
__device__ __forceinline__ float sum_same(int id, float v, int k, bool& first) {
    float sum = 0.f;
    first = id >= 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int idj = __shfl_sync(0xFFFFFFFFu, id, j, 8);
        const float vj = __shfl_sync(0xFFFFFFFFu, v, j, 8);
        if (idj == id) { sum += vj; first = first && j >= k; }
    }
    return sum;
}

template <int MODE>
__global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradParams p) {
    const unsigned FULL = 0xFFFFFFFFu;
    const int lane = threadIdx.x & 31, k = lane & 7;
    const int t0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 4, t = t0 + (lane >> 3);
    pdl_wait();
    if (t0 < p.T) {
        const Pick a = MODE == RG_TOPK ? Pick{-1, -INFINITY, 0.f} : load_pick(p, t, k, MODE != RG_DEEPSEEK);
        float4* zeros = reinterpret_cast<float4*>(p.d_logits + (size_t)t0 * p.E);
        for (int c = lane; c < min(4, p.T - t0) * (p.E >> 2); c += 32) zeros[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (MODE != RG_TOPK) {
            float weight = 0.f, slope = 0.f, g = 0.f;              // share of the pick, derivative of the sigmoid
            if (MODE == RG_DEEPSEEK || MODE == RG_LLAMA4) {
                const float e = expf(-fabsf(a.x)), inv = __fdiv_rn(1.0f, 1.0f + e);
                if (a.id >= 0) { weight = a.x >= 0.f ? inv : e * inv; slope = e * inv * inv; }
            } else {
                float mx = a.x;
#pragma unroll
                for (int off = 4; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
                if (a.id >= 0) weight = expf(a.x - mx);
            }
            if (MODE == RG_LLAMA4) {
                g = p.factor * a.d * slope;
            } else {
                float total = 0.f, diff = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float wj = __shfl_sync(FULL, weight, j, 8), dj = __shfl_sync(FULL, a.d, j, 8);
                    total += wj; diff = fmaf(a.d - dj, wj, diff);
                }
                if (MODE == RG_DEEPSEEK) {
                    total += 1e-20f; diff = fmaf(1e-20f, a.d, diff);
                    g = p.factor * __fdiv_rn(slope, total) * __fdiv_rn(diff, total);
                } else if (a.id >= 0) {
                    g = p.factor * __fdiv_rn(weight, total) * __fdiv_rn(diff, total);
                }
            }
            bool first;
            g = sum_same(a.id, g, k, first);
            __syncwarp();                                          // the rows' zeros are stored before the picks'
            if (first) p.d_logits[(size_t)t * p.E + a.id] = g;
        }
    }
    pdl_launch();
}

// The default form: one token per warp, every lane has COLS groups of four columns of its row, 128 columns apart.
template <int COLS>
__global__ void __launch_bounds__(256) route_grad_softmax_kernel(const RouteGradParams p) {
    const unsigned FULL = 0xFFFFFFFFu;
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    if (t < p.T) {
        const Pick a = load_pick(p, t, lane, true);                // (lanes behind top_k hold none)
        const float* logits = p.logits + (size_t)t * p.E;
        float* row = p.d_logits + (size_t)t * p.E;
        float z[COLS][4], mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < COLS; ++q) {
            const int c = q * 128 + lane * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) z[q][i] = -INFINITY;
            if (c < p.E) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(logits + c));
                z[q][0] = v.x; z[q][1] = v.y; z[q][2] = v.z; z[q][3] = v.w;
                if (p.bias)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[q][i] = __fadd_rn(z[q][i], __bfloat162float(p.bias[c + i]));
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, z[q][i]);
            }
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
        bool first;
        const float d_all = sum_same(a.id, a.d, lane, first);      // (of an expert picked twice only the first lane goes on)
        first = first && lane < 8;
        const float d = first ? d_all : 0.f, e = first ? expf(a.x - mx) : 0.f;
        unsigned mine = 0;                                         // the picked ones among this lane's columns
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int id = __shfl_sync(FULL, a.id, j);
            if (id >= 0 && (id & 127) >> 2 == lane) mine |= 1u << ((id >> 7) * 4 + (id & 3));
        }
        float rest = 0.f;                                          // of the experts that nobody picked
#pragma unroll
        for (int q = 0; q < COLS; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[q][i] = expf(z[q][i] - mx);
                if (!(mine >> (q * 4 + i) & 1u)) rest += z[q][i];
            }
#pragma unroll
        for (int off = 16; off; off >>= 1) rest += __shfl_xor_sync(FULL, rest, off);
        float others = rest, weighed = 0.f, total = rest, all = 0.f;       // without this lane's pick, and with all of them
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float ej = __shfl_sync(FULL, e, j), dj = __shfl_sync(FULL, d, j);
            total += ej; all = fmaf(ej, dj, all);
            if (j != lane) { others += ej; weighed = fmaf(ej, dj, weighed); }
        }
        const float inv = __fdiv_rn(1.0f, total);
        const float g = p.factor * (e * inv) * (d * (others * inv) - weighed * inv);
        const float back = -p.factor * (all * inv) * inv;
#pragma unroll
        for (int q = 0; q < COLS; ++q) {
            const int c = q * 128 + lane * 4;
            if (c < p.E) *reinterpret_cast<float4*>(row + c) = make_float4(z[q][0] * back, z[q][1] * back, z[q][2] * back, z[q][3] * back);
        }
        __syncwarp();                                              // the row is stored before the picks' gradients
        if (first) row[a.id] = g;
    }
    pdl_launch();
}

}  // namespace b200moe
