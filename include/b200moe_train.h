/*
 * b200moe_train.h -- C ABI of the training operators of libb200moe (sm_100a): what stands between the two GEMMs of an MoE
 * layer and around its router, with gradients.
 *
 * These entry points take no handle and keep no state: sizes are arguments, every launch goes to the caller's stream on the
 * current device, nothing is allocated, the host is not synchronised, and calls on different streams share nothing but what
 * the caller passes to both.  Return values as in b200moe.h.
 *
 * T tokens with top_k picks each (top_k <= 8, T * top_k <= 2^30); pair i = t * top_k + k; num_local experts (<= 512); hidden and
 * intermediate are multiples of 128 up to 2^20, row tensors have up to 2^30 rows.  All data pointers are device pointers; inputs are not modified, outputs overlap neither inputs
 * nor each other.  Row tensors have one of the three types below and start at a multiple of 32 bytes, e4m3 tensors at 16.  Sums
 * are fp32 in a fixed order with one rounding: results are the same from run to run.
 * (No counterpart in the reference, which has no backward pass.)
 */
#ifndef B200MOE_TRAIN_H_
#define B200MOE_TRAIN_H_

#include "b200moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200MOE_TYPE_BF16 0
#define B200MOE_TYPE_FP16 1
#define B200MOE_TYPE_FP32 2

/* Expert-sorted tables: the pairs whose expert topk_idx[i] - local_offset lies in [0, num_local) get one row each, the pairs of an expert
 * in ascending order (an expert picked twice by a token: two rows), every expert's segment padded to a multiple of `align` rows (a power of
 * two <= 128; b200moe_forward's own tables use 16).
 *   expert_row0 int32 [num_local + 1]  first row of each expert; the last entry is the number of rows in use
 *   row_pair    int32 [max_rows]       pair of a row, -1 for padding and behind the last segment
 *   pair_row    int32 [T, top_k]       row of a pair, -1 where it has none
 * max_rows >= T * top_k + (align - 1) * num_local holds every case.  With less, pairs whose row would lie behind it get none (as if
 * their expert were elsewhere), and expert_row0 ends at max_rows.
 * workspace: b200moe_sort_workspace_bytes(T, top_k, num_local) bytes, 16-byte aligned (none for up to 2048 pairs).  That is enough for every call with
 * no more pairs (T * top_k) and no more local experts.  It depends on the number of SMs of the device that is current: ask with the device current
 * that sorts. */
int b200moe_sort_workspace_bytes(int num_tokens, int top_k, int num_local, size_t* bytes);
int b200moe_sort_tokens(const int32_t* topk_idx, int num_tokens, int top_k, int num_local, int local_offset, int align, int max_rows,
                        int32_t* expert_row0, int32_t* row_pair, int32_t* pair_row, void* workspace, size_t workspace_bytes,
                        void* cuda_stream);

/* rows[r, :] = x[t, :] for every row r of a pair of token t, zeros in a segment's padding; rows behind expert_row0[num_local] are left as
 * they were.  x [T, hidden], rows [num_rows, hidden], of one type.  Its gradient is b200moe_combine without weights.
 * Indices outside their range in any table are treated like -1. */
int b200moe_permute(const void* x, int type, const int32_t* expert_row0, const int32_t* row_pair, const int32_t* pair_row,
                    int num_tokens, int top_k, int num_local, int hidden, int num_rows, void* rows, void* cuda_stream);

/* The same from activations that are kept in 8 bits: rows[r, :] = q[t, :] * scale[:, t], q and scale as b200moe_quantize_1x128 makes them
 * (e4m3 [T, hidden], float [hidden / 128, T]), rounded once to `type`.  With all three tables NULL row t is token t (T rows;
 * top_k, num_local and num_rows are not looked at). */
int b200moe_restore_1x128(const void* q_e4m3, const float* scale, int type, const int32_t* expert_row0, const int32_t* row_pair,
                          const int32_t* pair_row, int num_tokens, int top_k, int num_local, int hidden, int num_rows, void* rows,
                          void* cuda_stream);

/* out[t, :] = sum over k of topk_w[t, k] * rows[pair_row[t, k], :] in ascending k, pairs without a row left out; topk_w float [T, top_k], NULL =
 * ones (the gradient of b200moe_permute).  Every row of out [T, hidden] is written. */
int b200moe_combine(const void* rows, int type, const float* topk_w, const int32_t* pair_row, int num_tokens, int top_k, int hidden,
                    int num_rows, void* out, void* cuda_stream);

/* Gradients of b200moe_combine: grad_rows[r, :] = topk_w * grad_out[t, :] (zeros in padding, nothing behind the last segment) and
 * grad_w[t, k] = sum over columns of grad_out[t, :] * rows[r, :], float [T, top_k], zero for pairs without a row.
 * grad_rows must not overlap rows or grad_out. */
int b200moe_combine_backward(const void* grad_out, const void* rows, int type, const float* topk_w, const int32_t* expert_row0,
                             const int32_t* row_pair, const int32_t* pair_row, int num_tokens, int top_k, int num_local, int hidden,
                             int num_rows, void* grad_rows, float* grad_w, void* cuda_stream);

/* SwiGLU of GEMM1's rows [num_rows, 2 * intermediate] (columns as the operator has them: act = rows[:, :I] * silu(rows[:, I:])), and the 8-bit
 * copy of the rows that the backward pass works from: q e4m3 [num_rows, 2I], scale float [2I / 128, num_rows], scale = the smallest
 * power of two not below amax / 448 of the 128 columns (at least 2^-126; 1 where all are zero; NaN where one is infinite or NaN;
 * codes end at 240 under the scale 2^120: a finite value is restored as a finite one in fp32 and bf16; in fp16 one above 63488 is restored as an infinity).
 * used_rows: device pointer to the number of rows in use (expert_row0 + num_local), NULL = all; the others are left as they were.  Padding of the segments
 * is in use: it is taken like any row here and in the gradient, zeros give zeros, and what is not finite there stays so - the GEMMs around have to
 * leave zeros in it.  The sigmoid of a gate below -87 leaves fp32's
 * normal range and counts as zero, here and in the gradient (fp32 rows: it loses bits down to -88.7 and is zero below). */
int b200moe_swiglu_save(const void* gemm1_rows, int type, const int32_t* used_rows, int num_rows, int intermediate, void* act,
                        void* q_e4m3, float* scale, void* cuda_stream);

/* Its gradient from that copy: with up, gate = q * scale and s = sigmoid(gate), grad_gemm1_rows = [grad_act * gate * s |
 * grad_act * up * s * (1 + gate * (1 - s))], and, where `act` is not NULL, act = up * gate * s again (GEMM2's weight gradient needs it).
 * grad_act, grad_gemm1_rows and act have the one type. */
int b200moe_swiglu_backward(const void* q_e4m3, const float* scale, const void* grad_act, int type, const int32_t* used_rows,
                            int num_rows, int intermediate, void* grad_gemm1_rows, void* act, void* cuda_stream);

/* Gradient of b200moe_route's weights down to the logits: grad_logits float [T, E] from grad_w float [T, top_k], for the picks topk_idx that
 * b200moe_route made with the same logits, bias, factor and mode.  Every entry is written; ids outside [0, E) carry no weight, an expert
 * named twice in a row gets the sum.  num_experts a multiple of 32, <= 512; routing_logits and grad_logits 16-byte aligned.  In modes 1 to 5 the
 * bias is added to the logits, so its gradient is the column sum of grad_logits; in mode 0 it only selects and has none. */
int b200moe_route_backward(const float* routing_logits, const void* routing_bias, const int32_t* topk_idx, const float* grad_w,
                           int num_tokens, int num_experts, int top_k, float routed_scaling_factor, int routing_mode,
                           float* grad_logits, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* B200MOE_TRAIN_H_ */
