// Gradient of the routing weights down to the logits, one warp per token.  Lane k < top_k holds pick k: its expert, its logit and d = the
// gradient of its weight w (all sums over the token's picks; f = the routed scaling factor).
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
// The row of E logits is written once, zeros where nothing was picked; only the default form reads it whole.
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

constexpr int ROUTE_GRAD_COLS = 4;       // 128 columns each

template <int MODE>
__global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradParams p) {
    const unsigned FULL = 0xFFFFFFFFu;
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch();
    if (t >= p.T) return;
    float* row = p.d_logits + (size_t)t * p.E;
    const float* logits = p.logits + (size_t)t * p.E;
    int id = -1;
    float x = -INFINITY, d = 0.f;
    if (MODE != RG_TOPK && lane < p.top_k) {
        id = __ldg(p.topk_idx + (size_t)t * p.top_k + lane);
        if (id < 0 || id >= p.E) id = -1;
        if (id >= 0) {
            d = __ldg(p.d_w + (size_t)t * p.top_k + lane);
            x = __ldg(logits + id);
            if (MODE != RG_DEEPSEEK && p.bias) x = __fadd_rn(x, __bfloat162float(p.bias[id]));
        }
    }
    const unsigned same = __match_any_sync(FULL, id >= 0 ? id : -1 - lane);
    const bool first = id >= 0 && lane == __ffs(same) - 1;        // the lane that stores the expert's gradient
    float g = 0.f;
    if (MODE == RG_DEFAULT) {
        float z[ROUTE_GRAD_COLS][4], mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < ROUTE_GRAD_COLS; ++q) {
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
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
        // gradients of an expert picked twice are added; only its first lane goes on
        float sum = 0.f;
        for (int j = 0; j < p.top_k; ++j) {
            const float dj = __shfl_sync(FULL, d, j);
            if (same >> j & 1u) sum += dj;
        }
        d = first ? sum : 0.f;
        const float e = first ? expf(x - mx) : 0.f;
        unsigned mine = 0;                                         // the picked ones among this lane's columns
        for (int j = 0; j < p.top_k; ++j) {
            const int idj = __shfl_sync(FULL, id, j);
            if (idj >= 0 && (idj & 127) >> 2 == lane) mine |= 1u << ((idj >> 7) * 4 + (idj & 3));
        }
        float rest = 0.f;                                          // of the experts that nobody picked
#pragma unroll
        for (int q = 0; q < ROUTE_GRAD_COLS; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[q][i] = expf(z[q][i] - mx);
                if (!(mine >> (q * 4 + i) & 1u)) rest += z[q][i];
            }
        for (int off = 16; off; off >>= 1) rest += __shfl_xor_sync(FULL, rest, off);
        float others = rest, weighed = 0.f, total = rest, all = 0.f;       // without this lane's pick, and with all of them
        for (int j = 0; j < p.top_k; ++j) {
            const float ej = __shfl_sync(FULL, e, j), dj = __shfl_sync(FULL, d, j);
            total += ej; all = fmaf(ej, dj, all);
            if (j != lane) { others += ej; weighed = fmaf(ej, dj, weighed); }
        }
        const float inv = __fdiv_rn(1.0f, total);
        g = p.factor * (e * inv) * (d * (others * inv) - weighed * inv);
        const float back = -p.factor * (all * inv) * inv;
#pragma unroll
        for (int q = 0; q < ROUTE_GRAD_COLS; ++q) {
            const int c = q * 128 + lane * 4;
            if (c < p.E) *reinterpret_cast<float4*>(row + c) = make_float4(z[q][0] * back, z[q][1] * back, z[q][2] * back, z[q][3] * back);
        }
    } else {
        for (int c = lane * 4; c < p.E; c += 128) *reinterpret_cast<float4*>(row + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        if (MODE == RG_TOPK) return;
        float weight = 0.f, slope = 0.f;                           // share of the pick, derivative of the sigmoid
        if (MODE == RG_DEEPSEEK || MODE == RG_LLAMA4) {
            const float e = expf(-fabsf(x)), inv = __fdiv_rn(1.0f, 1.0f + e);
            if (id >= 0) { weight = x >= 0.f ? inv : e * inv; slope = e * inv * inv; }
        } else {
            float mx = x;
            for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
            if (id >= 0) weight = expf(x - mx);
        }
        if (MODE == RG_LLAMA4) {
            g = p.factor * d * slope;
        } else {
            float total = 0.f, diff = 0.f;
            for (int j = 0; j < p.top_k; ++j) {
                const float wj = __shfl_sync(FULL, weight, j), dj = __shfl_sync(FULL, d, j);
                total += wj; diff = fmaf(d - dj, wj, diff);
            }
            if (MODE == RG_DEEPSEEK) {
                total += 1e-20f; diff = fmaf(1e-20f, d, diff);
                g = p.factor * __fdiv_rn(slope, total) * __fdiv_rn(diff, total);
            } else if (id >= 0) {
                g = p.factor * __fdiv_rn(weight, total) * __fdiv_rn(diff, total);
            }
        }
        float sum = 0.f;
        for (int j = 0; j < p.top_k; ++j) {
            const float gj = __shfl_sync(FULL, g, j);
            if (same >> j & 1u) sum += gj;
        }
        g = sum;
    }
    __syncwarp();                                                  // the row's zeros are stored before the picks'
    if (first) row[id] = g;
}

}  // namespace b200moe
