/* Microscaled 4-bit matrices (MXFP4) and the dense layer over them.
 *
 * A row is cut into blocks of 32 elements. A block holds one power-of-two
 * scale 2^(s - 127) (E8M0 byte s) and 32 E2M1 codes: sign, two exponent bits,
 * one fraction bit, with the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6. With m the
 * block's largest magnitude,
 *   s = max(floor(log2 m) - 2, -127) + 127        (0 for a block of zeros)
 *   code = x / 2^(s - 127) rounded to the nearest magnitude, ties to the code
 *          with an even fraction bit, larger magnitudes to 6.
 * A block with an infinity or a NaN gets s = 255 (NaN) and zero codes: all
 * its elements stand for NaN, and so does every product that reads it. A row
 * whose length is no multiple of 32 ends in a shorter block.
 *
 * These layers stand beside xse_dlrm.h's; the reference's tower runs its
 * Dense layers in fp32 under XLA (examples/dlrm/model_jce.py:107-138) and has
 * no counterpart. All buffers are memory of the current device, outputs
 * without elements in common with inputs or the workspace; `stream` is a
 * cudaStream_t (NULL: the legacy default stream). Calls return after their
 * launches; status codes and xse_last_error() as in xse_emb.h. No call keeps
 * memory of its own, so calls on several streams or in captured graphs only
 * share what the caller lets them share.
 */
#ifndef XSE_MX_H_
#define XSE_MX_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* `groups` matrices of [rows, cols] in 4 bits (rows < 2^31, cols <= 2^30), as
 * one allocation each of codes and scales:
 *   codes: [groups][rows][16 * ceil(cols / 32)] bytes, element 2i in the low
 *          half of byte i; 16-byte aligned. Codes past the last column are 0
 *          (xse_mxfp4_quantize writes them).
 *   scales: [groups][ceil(rows / 128)][ceil(cols / 128)][512] bytes; block b
 *          of row r lies in tile (r / 128, b / 4) at byte
 *          (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4; 16-byte aligned.
 *          Bytes of blocks past the last one are 0; those of rows past the
 *          last one are not written and not used. */
typedef struct xse_mx_matrix {
  void* codes;
  void* scales;
  int64_t rows;
  int32_t cols;
  int32_t groups;
} xse_mx_matrix;

/* Bytes of the two buffers (0 for sizes that are not served: out of range, or of
 * 2^63 bytes or more). */
int64_t xse_mxfp4_codes_bytes(int64_t rows, int32_t cols, int32_t groups);
int64_t xse_mxfp4_scales_bytes(int64_t rows, int32_t cols, int32_t groups);

/* q = the quantisation of x, element (g, r, c) at x[g * group_stride +
 * r * row_stride + c * col_stride] (elements; any strides, so a layer's
 * [in, out] kernel is quantised as rows = out with row_stride 1). `dtype` is
 * XSE_DT_F32 or XSE_DT_BF16. */
int xse_mxfp4_quantize(const void* x, int32_t dtype, int64_t group_stride,
                       int64_t row_stride, int64_t col_stride,
                       const xse_mx_matrix* q, void* stream);

/* out = the values q stands for (exact in XSE_DT_F32 and XSE_DT_BF16 for the
 * scales that xse_mxfp4_quantize gives, up to 252; with 253 and 254 the largest
 * codes pass the types' range and give infinities), row r of group g at
 * out + g * group_stride + r * row_stride, row_stride >= cols. */
int xse_mxfp4_dequantize(const xse_mx_matrix* q, void* out, int32_t dtype,
                         int64_t group_stride, int64_t row_stride,
                         void* stream);

/* y = act(x W^T + bias) for quantised x (one group, [rows, in]) and w (one
 * group, [out, in]): products of the 4-bit values with their scales on the
 * tensor cores, accumulated in fp32, plus bias (fp32, [out] or NULL), act
 * (XSE_ACT_*), one rounding to y_dtype (XSE_DT_F32 or XSE_DT_BF16). Row r of y
 * at y + r * y_stride, y_stride >= out. */
int xse_linear_forward_mxfp4_q(const xse_mx_matrix* x, const xse_mx_matrix* w,
                               const float* bias, int32_t activation, void* y,
                               int32_t y_dtype, int64_t y_stride,
                               void* stream);

/* The same from unquantised x ([rows, in] of x_dtype, row stride x_stride),
 * which is quantised on the way: equal to xse_mxfp4_quantize followed by
 * xse_linear_forward_mxfp4_q. `workspace` holds
 * xse_linear_mxfp4_workspace(rows, in) bytes (none for a few rows: it may then
 * be NULL), 16-byte aligned, used until the call's work on `stream` is done. */
int64_t xse_linear_mxfp4_workspace(int64_t rows, int32_t in_dim);
int xse_linear_forward_mxfp4(const void* x, int32_t x_dtype, int64_t rows,
                             int64_t x_stride, const xse_mx_matrix* w,
                             const float* bias, int32_t activation, void* y,
                             int32_t y_dtype, int64_t y_stride,
                             void* workspace, int64_t workspace_bytes,
                             void* stream);

/* Waits for `stream` and reports whether a product's kernel on the current
 * device gave up one of its bounded waits since the last check
 * (DEADLINE_EXCEEDED; its outputs are then incomplete). Not for use while a
 * stream is being captured. */
int xse_mxfp4_check(void* stream);

#ifdef __cplusplus
}
#endif

#endif /* XSE_MX_H_ */
