// Host side of the training operators of libb200moe (token order, 8-bit SwiGLU copies, router gradient): argument checks and
// launches for the C ABI declared in include/b200moe_train.h.  Nothing here keeps state: every call works on its arguments alone, on
// the current device and the caller's stream, so calls on different streams share nothing.
#include <cuda_runtime.h>

#include "b200moe_train.h"
#include "order.cuh"
#include "route_grad.cuh"
#include "swiglu.cuh"

using namespace b200moe;

namespace {

// Launched with programmatic stream serialization: the start hides under the tail of the kernel before it, and every kernel waits for
// that one to complete before it reads or writes global memory.
template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, int block, void* stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, KArgs(args)...);
}

int sm_count() {
    const int n = b200moe_num_sms();
    return n > 0 ? n : 148;
}

bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

bool known_type(int type) { return type == B200MOE_TYPE_BF16 || type == B200MOE_TYPE_FP16 || type == B200MOE_TYPE_FP32; }
int type_bytes(int type) { return type == B200MOE_TYPE_FP32 ? 4 : 2; }

// Slices of a thread's one pair each, longer ones where that would be more CTAs than the chip holds at once (every CTA reads all slices'
// histograms).  Up to SORT_ALONE pairs one CTA and one launch: 2048 pairs 5.8 us against 5.5 (and 4 us less of host time), 4096: 9.3 against 5.5.
int sort_slice(int n) {
    const int most = 2 * sm_count();
    return ((n + most - 1) / most + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
}
int sort_ctas(int n) { return n <= SORT_ALONE ? 1 : (n + sort_slice(n) - 1) / sort_slice(n); }
size_t sort_bytes(int n, int num_local) {
    const int ctas = sort_ctas(n);
    return ctas > 1 ? (size_t)ctas * sort_pitch(num_local) * sizeof(int) : 0;
}
// What a caller is told: enough for this size and every smaller one.  (Slices grow by whole SORT_THREADS, so that the CTAs of a call, and with them
// sort_bytes, fall where a slice takes one pair per thread more: on 148 SMs 296 CTAs for 303104 pairs, 149 for 303112.)
size_t sort_bytes_upto(int n, int num_local) {
    const size_t ctas = n <= SORT_ALONE ? 0 : min((n + SORT_THREADS - 1) / SORT_THREADS, 2 * sm_count());
    return ctas * sort_pitch(num_local) * sizeof(int);
}

constexpr int MAX_COLUMNS = 1 << 20, MAX_ROWS = 1 << 30;      // (index arithmetic stays in range; far above what a GPU's memory holds)

bool bad_picks(int T, int top_k) { return T < 0 || top_k < 1 || top_k > ORDER_MAX_PICKS || (long long)T * top_k > (1ll << 30); }

// The sizes and tables that the row kernels share
int check_order(const OrderParams& o, int H) {
    if (bad_picks(o.T, o.top_k) || o.num_local < 1 || o.num_local > ORDER_MAX_LOCAL || o.num_rows < 0 || o.num_rows > MAX_ROWS || H <= 0 ||
        H % 128 || H > MAX_COLUMNS)
        return B200MOE_E_BADARG;
    return 0;
}

// CTAs that look through the padding of `rows` rows: a row a warp, as long as the chip holds them at once
long long padding_ctas(long long rows, int warps, int per_sm) { return min((rows + warps - 1) / warps, (long long)per_sm * sm_count()); }

// CTAs of a kernel whose threads take one unit of a token's row each.  Starting CTAs is what bounds a call that has little to do for each unit: plain
// rows read back from 8 bits, rows of which few have a place here.  Nothing is shared inside a CTA, so small ones are even where padding is most of the work.
// us, CTAs of 64 / 128 / 256 threads: 4096 x 7168 plain 31.5 / 17.8 / 18.0, 512 x 7168 plain 4.8 / 3.0 / 2.6; permute of 8192 tokens of 7168 columns on an eighth of
// the experts 61.6 / 38.9 / 40.3, of 1024 9.3 / 6.3 / 6.5, with every expert here level; 8192 x 128 on an eighth 4.6 / 3.2 / 3.3, with every expert 5.1 / 5.2 / 5.6.
// Few tokens of wide rows over 256 experts: 64 tokens 9.0 / 10.0 / 11.1, 128: 11.4 / 12.6 / 13.5; of 2048 columns 64 tokens 3.2 / 3.4 / 4.3, 256: 4.3 / 4.8 / 5.7, 1024 on
// an eighth 5.0 / 3.2 / 2.9; of 256 columns 256 tokens 4.0 / 2.3 / 2.7.  So 256 threads without padding, 64 for wide rows of few tokens (up to 12 CTAs per
// SM), 128 otherwise.
int unit_block(long long T, int units, long long pad_rows) {
    if (pad_rows == 0) return PERMUTE_THREADS;
    return units >= 128 && T * units <= 12ll * 64 * sm_count() ? 64 : 128;
}
int unit_grid(long long T, int units, long long pad_rows, int block) {
    return (int)min(max(max((T * units + block - 1) / block, padding_ctas(pad_rows, block / 32, 1536 / block)), 1ll), 1ll << 24);
}

template <typename T>
int combine_rows(const OrderParams& o, const void* rows, const float* w, void* out, int H, void* stream) {
    const long long units = (long long)o.T * (H * (int)sizeof(T) / 32);
    const int grid = (int)min((units + COMBINE_THREADS - 1) / COMBINE_THREADS, (long long)COMBINE_CTAS * sm_count());
    return launch(combine_rows_kernel<T>, dim3(grid), COMBINE_THREADS, stream, o, static_cast<const T*>(rows), w, static_cast<T*>(out), H);
}

template <typename T>
int combine_grad(const OrderParams& o, const void* d_out, const void* rows, const float* w, void* d_rows, float* d_w, int H, void* stream) {
    const int units = H * (int)sizeof(T) / 16;
    // by tokens: more than one warp where a thread would have more than four units, up to 128 threads; by rows: one warp, more for few tokens, whose rows do not fill the chip
    int token_sh = 5, row_sh = 5;
    while (token_sh < 7 && units > 4 << token_sh) ++token_sh;
    while (o.T <= 64 && row_sh < 7 && units >= 2 * GRAD_FLIGHT << row_sh) ++row_sh;
    const int tokens = GRAD_THREADS >> token_sh;
    const int grid = (int)max(max(min(((long long)o.T + tokens - 1) / tokens, 16ll * sm_count()), padding_ctas(o.num_rows, GRAD_WARPS, 4)), 1ll);
    return launch(combine_grad_kernel<T>, dim3(grid), GRAD_THREADS, stream, o, static_cast<const T*>(d_out), static_cast<const T*>(rows), w,
                  static_cast<T*>(d_rows), d_w, H, token_sh, row_sh);
}

template <typename T>
int restore_rows(const OrderParams& o, const void* q, const float* scale, void* rows, int H, void* stream) {
    const int units = H / 16, pad_rows = o.pair_row ? o.num_rows : 0, block = unit_block(o.T, units, pad_rows);
    return launch(restore_rows_kernel<T>, unit_grid(o.T, units, pad_rows, block), block, stream, o, static_cast<const uint8_t*>(q), scale,
                  static_cast<T*>(rows), H);
}

// Block of a CTA of the SwiGLU kernels, 2^rsh rows of gpc pairs of groups; less where that leaves few CTAs per SM.
// save: the fewest rows, two at least (scales leave as runs of rows), that keep the CTA's threads busy in four fifths of its turns.  One / two / four rows
// of 2048 columns, us: 2000 rows 6.7 / 6.3 / 8.3, 34645: 90.2 / 87.8 / 88.8; four / eight / 16 of 640 columns (five groups: 62, 83 and 100 %) 40000 rows
// 38.8 / 35.7 / 37.4; four / eight / 16 of 256 columns 20000 rows 11.8 / 9.2 / 9.8.  Under four CTAs per SM a block of several turns is halved, first its
// rows, then its groups: 2000 rows of 640 columns 3.1 (fp32 4.4) against 3.4 (5.4) for a line at two CTAs, 1000 of 2048 fp32 5.5 against 6.6, 5000 of 384 fp32 6.5 against 8.2.
// A block of one turn stays whole: halves leave threads idle (500 rows of 128 columns 1.9 against 2.2).
// (256 threads per CTA: level for 2048 columns, 93.5 against 91.9 under the clocks of a long run, 40000 x 640 37.8, 20000 x 256 9.6.)
// backward: nothing is kept between turns, so about one turn: two / four / eight rows of 2048 columns 8000 rows 26.7 / 27.4 / 28.2, 34645: 106.0 / 108.3 /
// 110.6; four / eight / 16 of 640 columns 40.0 / 41.2 / 42.2; eight / 16 of 256 columns 20000 rows 10.1 / 10.2.  (fp32 rows: two / four of 2048 columns 194 / 190,
// of 1536 155 / 143.  128 threads per CTA with half the rows: level, 109.6 against 108.1 in a long run.)
void swiglu_block(bool save, int rows, int I, int& rsh, int& gpc, dim3& grid) {
    const int groups = I >> 7;
    int parts = (groups + 63) / 64;
    gpc = (groups + parts - 1) / parts;
    auto ctas = [&] { return (long long)((rows + (1 << rsh) - 1) >> rsh) * parts; };
    if (save) {
        for (rsh = 1; rsh < 5 && (gpc << (rsh + 1)) <= SWIGLU_SCALES; ++rsh) {
            const int items = gpc << rsh, turns = (items + SAVE_TURN - 1) / SAVE_TURN;
            if (items * 5 >= turns * SAVE_TURN * 4) break;
        }
        while ((gpc << rsh) > SAVE_TURN && ctas() < 4ll * sm_count()) {
            if (rsh > 0) --rsh;
            else { ++parts; gpc = (groups + parts - 1) / parts; }
        }
    } else {
        for (rsh = 0; rsh < 5 && (gpc << rsh) * 8 < GRAD_X_TURN * 5; ++rsh) {}
        while (rsh > 0 && ctas() < 2ll * sm_count()) --rsh;
    }
    grid = dim3((rows + (1 << rsh) - 1) >> rsh, (groups + gpc - 1) / gpc);
}

template <typename T>
int swiglu_save(const void* x, const int32_t* used, int rows, int I, void* act, void* q, float* scale, void* stream) {
    int rsh, gpc;
    dim3 grid;
    swiglu_block(true, rows, I, rsh, gpc, grid);
    return launch(swiglu_save_kernel<T>, grid, SAVE_THREADS, stream, static_cast<const T*>(x), used, rows, I, rsh, gpc, static_cast<T*>(act),
                  static_cast<uint8_t*>(q), scale);
}

template <typename T>
int swiglu_grad(const void* q, const float* scale, const void* d_act, const int32_t* used, int rows, int I, void* d_x, void* act, void* stream) {
    int rsh, gpc;
    dim3 grid;
    swiglu_block(false, rows, I, rsh, gpc, grid);
    return launch(act ? swiglu_grad_kernel<T, true> : swiglu_grad_kernel<T, false>, grid, GRAD_X_THREADS, stream, static_cast<const uint8_t*>(q), scale,
                  static_cast<const T*>(d_act), used, rows, I, rsh, gpc, static_cast<T*>(d_x), static_cast<T*>(act));
}

}  // namespace

#define BY_TYPE(call) (type == B200MOE_TYPE_BF16 ? call<__nv_bfloat16> : type == B200MOE_TYPE_FP16 ? call<__half> : call<float>)

extern "C" {

int b200moe_sort_workspace_bytes(int T, int top_k, int num_local, size_t* bytes) {
    if (!bytes || bad_picks(T, top_k) || num_local < 1 || num_local > ORDER_MAX_LOCAL) return B200MOE_E_BADARG;
    *bytes = sort_bytes_upto(T * top_k, num_local);
    return 0;
}

int b200moe_sort_tokens(const int32_t* topk_idx, int T, int top_k, int num_local, int local_offset, int align, int max_rows,
                        int32_t* expert_row0, int32_t* row_pair, int32_t* pair_row, void* workspace, size_t workspace_bytes, void* stream) {
    if (bad_picks(T, top_k) || num_local < 1 || num_local > ORDER_MAX_LOCAL || align < 1 || align > 128 || (align & (align - 1)) || max_rows < 0 ||
        max_rows > MAX_ROWS)
        return B200MOE_E_BADARG;
    if (!expert_row0 || (max_rows && !row_pair) || (T && (!topk_idx || !pair_row))) return B200MOE_E_BADARG;
    SortParams p;
    p.topk_idx = topk_idx; p.n = T * top_k; p.num_local = num_local; p.local_offset = local_offset; p.align = align; p.max_rows = max_rows;
    p.slices = static_cast<int*>(workspace); p.expert_row0 = expert_row0; p.row_pair = row_pair; p.pair_row = pair_row;
    p.slice = max(sort_slice(p.n), SORT_THREADS);
    const int ctas = sort_ctas(p.n);
    if (ctas == 1) return launch(sort_one_kernel, dim3(1), SORT_THREADS, stream, p);
    if (!workspace || misaligned(workspace, 16) || workspace_bytes < sort_bytes(p.n, num_local)) return B200MOE_E_WORKSPACE;
    const int rc = launch(sort_count_kernel, dim3(ctas), SORT_THREADS, stream, p);
    return rc ? rc : launch(sort_place_kernel, dim3(ctas), SORT_THREADS, stream, p);
}

int b200moe_permute(const void* x, int type, const int32_t* expert_row0, const int32_t* row_pair, const int32_t* pair_row, int T, int top_k,
                    int num_local, int hidden, int num_rows, void* rows, void* stream) {
    const OrderParams o = {expert_row0, row_pair, pair_row, T, top_k, num_local, num_rows};
    if (!known_type(type) || check_order(o, hidden)) return B200MOE_E_BADARG;
    if (num_rows == 0) return 0;
    if (!expert_row0 || !row_pair || !rows || (T && (!x || !pair_row)) || misaligned(x, 32) || misaligned(rows, 32)) return B200MOE_E_BADARG;
    const int units = hidden * type_bytes(type) / 32, block = unit_block(T, units, num_rows);
    return launch(permute_rows_kernel, unit_grid(T, units, num_rows, block), block, stream, o, static_cast<const char*>(x), static_cast<char*>(rows), units);
}

int b200moe_restore_1x128(const void* q, const float* scale, int type, const int32_t* expert_row0, const int32_t* row_pair, const int32_t* pair_row,
                          int T, int top_k, int num_local, int hidden, int num_rows, void* rows, void* stream) {
    const OrderParams o = {expert_row0, row_pair, pair_row, T, top_k, num_local, num_rows};
    if (!known_type(type) || misaligned(q, 16) || misaligned(rows, 32)) return B200MOE_E_BADARG;
    if (pair_row || row_pair || expert_row0) {
        if (check_order(o, hidden)) return B200MOE_E_BADARG;
        if (num_rows == 0) return 0;
        if (!expert_row0 || !row_pair || !rows || (T && (!q || !scale || !pair_row))) return B200MOE_E_BADARG;
    } else {
        if (T < 0 || T > MAX_ROWS || hidden <= 0 || hidden % 128 || hidden > MAX_COLUMNS) return B200MOE_E_BADARG;
        if (T == 0) return 0;
        if (!q || !scale || !rows) return B200MOE_E_BADARG;
    }
    return BY_TYPE(restore_rows)(o, q, scale, rows, hidden, stream);
}

int b200moe_combine(const void* rows, int type, const float* topk_w, const int32_t* pair_row, int T, int top_k, int hidden, int num_rows, void* out,
                    void* stream) {
    const OrderParams o = {nullptr, nullptr, pair_row, T, top_k, 1, num_rows};
    if (!known_type(type) || check_order(o, hidden)) return B200MOE_E_BADARG;
    if (T == 0) return 0;
    if (!pair_row || !out || (num_rows && !rows) || misaligned(rows, 32) || misaligned(out, 32)) return B200MOE_E_BADARG;
    return BY_TYPE(combine_rows)(o, rows, topk_w, out, hidden, stream);
}

int b200moe_combine_backward(const void* grad_out, const void* rows, int type, const float* topk_w, const int32_t* expert_row0, const int32_t* row_pair,
                             const int32_t* pair_row, int T, int top_k, int num_local, int hidden, int num_rows, void* grad_rows, float* grad_w,
                             void* stream) {
    const OrderParams o = {expert_row0, row_pair, pair_row, T, top_k, num_local, num_rows};
    if (!known_type(type) || check_order(o, hidden)) return B200MOE_E_BADARG;
    if (T == 0 && num_rows == 0) return 0;
    if (!expert_row0 || (num_rows && (!row_pair || !rows || !grad_rows)) || (T && (!grad_out || !topk_w || !pair_row || !grad_w))) return B200MOE_E_BADARG;
    if (misaligned(grad_out, 32) || misaligned(rows, 32) || misaligned(grad_rows, 32)) return B200MOE_E_BADARG;
    return BY_TYPE(combine_grad)(o, grad_out, rows, topk_w, grad_rows, grad_w, hidden, stream);
}

int b200moe_swiglu_save(const void* gemm1_rows, int type, const int32_t* used_rows, int num_rows, int intermediate, void* act, void* q, float* scale,
                        void* stream) {
    if (!known_type(type) || num_rows < 0 || num_rows > MAX_ROWS || intermediate <= 0 || intermediate % 128 || intermediate > MAX_COLUMNS)
        return B200MOE_E_BADARG;
    if (num_rows == 0) return 0;
    if (!gemm1_rows || !act || !q || !scale || misaligned(gemm1_rows, 32) || misaligned(act, 32) || misaligned(q, 16)) return B200MOE_E_BADARG;
    return BY_TYPE(swiglu_save)(gemm1_rows, used_rows, num_rows, intermediate, act, q, scale, stream);
}

int b200moe_swiglu_backward(const void* q, const float* scale, const void* grad_act, int type, const int32_t* used_rows, int num_rows, int intermediate,
                            void* grad_gemm1_rows, void* act, void* stream) {
    if (!known_type(type) || num_rows < 0 || num_rows > MAX_ROWS || intermediate <= 0 || intermediate % 128 || intermediate > MAX_COLUMNS)
        return B200MOE_E_BADARG;
    if (num_rows == 0) return 0;
    if (!q || !scale || !grad_act || !grad_gemm1_rows) return B200MOE_E_BADARG;
    if (misaligned(q, 16) || misaligned(grad_act, 32) || misaligned(grad_gemm1_rows, 32) || misaligned(act, 32)) return B200MOE_E_BADARG;
    return BY_TYPE(swiglu_grad)(q, scale, grad_act, used_rows, num_rows, intermediate, grad_gemm1_rows, act, stream);
}

int b200moe_route_backward(const float* routing_logits, const void* routing_bias, const int32_t* topk_idx, const float* grad_w, int T, int num_experts,
                           int top_k, float routed_scaling_factor, int routing_mode, float* grad_logits, void* stream) {
    if (bad_picks(T, top_k) || num_experts < 32 || num_experts > ROUTE_GRAD_MAX || num_experts % 32 || top_k > num_experts) return B200MOE_E_BADARG;
    if (routing_mode < 0 || routing_mode >= RG_COUNT || (routing_mode == RG_LLAMA4 && top_k != 1)) return B200MOE_E_BADARG;
    if (T == 0) return 0;
    if (!routing_logits || !topk_idx || !grad_w || !grad_logits || misaligned(routing_logits, 16) || misaligned(grad_logits, 16)) return B200MOE_E_BADARG;
    const RouteGradParams p = {routing_logits, static_cast<const __nv_bfloat16*>(routing_bias), topk_idx, grad_w, grad_logits, T, num_experts, top_k,
                               routed_scaling_factor};
    if (routing_mode == RG_DEFAULT) {
        auto* kern = num_experts <= 128 ? route_grad_softmax_kernel<1> : num_experts <= 256 ? route_grad_softmax_kernel<2> : route_grad_softmax_kernel<4>;
        return launch(kern, dim3((T + 7) / 8), 256, stream, p);
    }
    auto* kern = routing_mode == RG_DEEPSEEK ? route_grad_kernel<RG_DEEPSEEK>
                 : routing_mode == RG_LLAMA4 ? route_grad_kernel<RG_LLAMA4>
                 : routing_mode == RG_TOPK   ? route_grad_kernel<RG_TOPK>
                                             : route_grad_kernel<RG_RENORMALIZE>;
    return launch(kern, dim3((T + 31) / 32), 256, stream, p);
}

}  // extern "C"
