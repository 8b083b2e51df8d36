/* Rows sorted by expert and back, and the experts' 4-bit dense layers.
 *
 * A router gives each of `tokens` rows `topk` experts: pair p = t * topk + j
 * is row t's j-th choice. xse_expert_sort orders the pairs by expert; the
 * other calls move rows between the tokens' order and the sorted one:
 *   offsets [num_experts + 1]: expert e's sorted rows are
 *                              [offsets[e], offsets[e + 1])
 *   order [tokens * topk]:     the pair of each sorted row, -1 behind the last
 *   slots [tokens * topk]:     the sorted row of each pair, -1 for a dropped
 *                              one
 * all int32. Pairs of one expert keep their order. A pair whose id lies
 * outside [0, num_experts) is dropped: the padding rows of a batch are given
 * -1. Rows behind the last sorted row are written with zeros.
 *
 * The combination is a weighted-sum bag over the sorted rows (xse_emb.h pools
 * such bags from tables); the reference has no counterpart. Buffers, streams
 * and status codes as in xse_mx.h. Values are float32 or bfloat16
 * (XSE_DT_F32, XSE_DT_BF16), weights float32; sums are fp32 in the order of
 * the choices, rounded once. Row strides are in elements.
 */
#ifndef XSE_EXPERTS_H_
#define XSE_EXPERTS_H_

#include <stdint.h>

#include "xse_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

#define XSE_MAX_EXPERTS 1024

typedef struct xse_expert_plan {
  int32_t* offsets;
  int32_t* order;
  int32_t* slots;
  int64_t tokens;
  int32_t topk;
  int32_t num_experts;
} xse_expert_plan;

/* Fills the plan's three arrays from ids [tokens, topk] (ids_type
 * XSE_INDEX_I32 or XSE_INDEX_I64, contiguous). tokens * topk < 2^31 and
 * 1 <= num_experts <= XSE_MAX_EXPERTS. `workspace` holds
 * xse_expert_sort_workspace(tokens * topk, num_experts) bytes (none for small
 * batches: it may then be NULL), 4-byte aligned, used until the call's work on
 * `stream` is done. */
int64_t xse_expert_sort_workspace(int64_t pairs, int32_t num_experts);
int xse_expert_sort(const void* ids, int32_t ids_type,
                    const xse_expert_plan* plan, void* workspace,
                    int64_t workspace_bytes, void* stream);

/* out[r] = x[order[r] / topk] for every sorted row r, zeros behind the last:
 * x [tokens, cols], out [tokens * topk, cols]. Its gradient is
 * xse_expert_combine without weights. */
int xse_expert_gather(const void* x, int32_t dtype, int32_t cols,
                      int64_t x_stride, const xse_expert_plan* plan, void* out,
                      int64_t out_stride, void* stream);

/* out[t] = sum over j of weights[t, j] * y[slots[t, j]] (weights [tokens,
 * topk], or NULL for 1), dropped pairs left out; a row without pairs is zero. */
int xse_expert_combine(const void* y, int32_t dtype, int32_t cols,
                       int64_t y_stride, const xse_expert_plan* plan,
                       const float* weights, void* out, int64_t out_stride,
                       void* stream);

/* The gradients of xse_expert_combine for grad [tokens, cols]:
 *   grad_y[r] = weights[order[r]] * grad[order[r] / topk], zeros behind the
 *               last sorted row
 *   grad_weights[t, j] = sum over c of grad[t, c] * y[slots[t, j], c], 0 for
 *               a dropped pair
 * Either output may be NULL, with grad_weights NULL y may be too; weights may
 * be NULL (1). */
int xse_expert_combine_backward(const void* grad, const void* y, int32_t dtype,
                                int32_t cols, int64_t grad_stride,
                                int64_t y_stride, const xse_expert_plan* plan,
                                const float* weights, void* grad_y,
                                int64_t grad_y_stride, float* grad_weights,
                                void* stream);

/* y[r] = act(x_r W_e^T + bias_e) for every sorted row r of expert e, zeros
 * behind the last: xse_linear_forward_mxfp4 with w [num_experts] groups of
 * [out, in] and bias [num_experts, out] or NULL. With `sorted` 0, x is
 * [tokens, in] and x_r is row order[r] / topk; with 1, x is
 * [tokens * topk, in] in sorted order (another such layer's output) and rows
 * behind the last do not matter. y is [tokens * topk, out]. `workspace` as
 * xse_linear_forward_mxfp4's. */
int64_t xse_expert_linear_workspace(int64_t pairs, int32_t num_experts,
                                    int32_t in_dim);
int xse_expert_linear_mxfp4(const void* x, int32_t x_dtype, int64_t x_stride,
                            int32_t sorted, const xse_expert_plan* plan,
                            const xse_mx_matrix* w, const float* bias,
                            int32_t activation, void* y, int32_t y_dtype,
                            int64_t y_stride, void* workspace,
                            int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* XSE_EXPERTS_H_ */
