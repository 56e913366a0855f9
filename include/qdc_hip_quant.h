/* qdc_hip_quant.h -- entry points of libqdc_hip.so for projections whose weights are held
 * in 4 bits and whose input rows may be held in 8.  Types, status codes, dtype codes and
 * stream rules are those of qdc_hip.h: nothing is allocated or kept, everything is
 * enqueued on `stream`, and a negative status is returned before anything is enqueued.
 * The reference keeps every weight in fp32 or bf16 and has no counterpart of these.
 *
 * A weight [out, inner] in 4 bits: value = q * s, q a whole number of -8..7, s a bf16
 * scale for each output and group of `group` (32, 64 or 128) inputs.  Held as blocks of
 * 16 outputs by 128 inputs, nb = ceil(out / 16) by kb = ceil(inner / 128) of them:
 *   packed  int32 [nb, kb, 64, 4]: word t of lane l holds the inputs 32 t + 8 (l / 16) +
 *           0..7 of the block, of its output l % 16: input j < 4 in bits 8 j .. 8 j + 3,
 *           input 4 + j in bits 8 j + 4 .. 8 j + 7, two's complement;
 *   scales  bf16 [nb, kb * 128 / group, 16].
 * What lies behind the last output and input is 0.  inner is a multiple of 8.  A gated
 * weight is two of out / 2 outputs, gate and up, whose blocks alternate (nb is twice
 * ceil(out / 2 / 16)): block 2 j is gate's block j, block 2 j + 1 up's.
 *
 * Rows in 8 bits (QDC_Q8): value = i * a, i int8 [rows, width] of -127..127, a fp32 [rows,
 * ceil(width / 128)], a scale for each 128 columns; width is a multiple of 16.  A group of
 * zeros has a = 0; one that holds an infinity or a NaN has it as a: its values are NaN.
 * Pointers are 16-byte aligned, scales of 8-bit rows 4-byte aligned (QDC_ERR_SHAPE
 * otherwise); outputs overlap neither each other nor an input (QDC_ERR_ALIAS).
 */
#ifndef QDC_HIP_QUANT_H
#define QDC_HIP_QUANT_H

#include "qdc_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header, and of the library that was built with it; the minor number
 * changes with a signature, the patch number with added entry points. */
#define QDC_HIP_QUANT_VERSION "qdc_hip_quant 0.1.0"
const char *qdc_quant_version(void);

#define QDC_Q8 3 /* rows in 8 bits with scales, beside the dtype codes of qdc_hip.h */

/* packed and scales of w [out, inner] (fp32 or bf16, rows ld elements apart, a multiple of
 * 8): s = bf16(max |w| / 7) of each group, q = w / s rounded to nearest even, within -7..7.
 * A group whose s is 0 has q = 0; one that holds an infinity or a NaN has s = NaN.
 * gated != 0: w is [gate; up], out even. */
int32_t qdc_pack_w4(void *packed, void *scales, const void *w, int64_t out, int64_t inner,
                    int64_t ld, int64_t group, int32_t gated, int32_t dtype, hipStream_t stream);

/* w [out, inner] contiguous (fp32, or bf16: rounded to nearest even) from packed and scales. */
int32_t qdc_unpack_w4(void *w, const void *packed, const void *scales, int64_t out, int64_t inner,
                      int64_t group, int32_t gated, int32_t dtype, hipStream_t stream);

/* Rows x [rows, width] (fp32 or bf16, ld elements apart, a multiple of 8) in 8 bits: a = max
 * |x| / 127 of each group, in fp32, i = x / a rounded to nearest even, within -127..127. */
int32_t qdc_quantize_q8(void *q, float *scales, const void *x, int64_t rows, int64_t width,
                        int64_t ld, int32_t dtype, hipStream_t stream);

/* out [rows, width] contiguous (fp32, or bf16: rounded to nearest even) from rows in 8 bits. */
int32_t qdc_dequantize_q8(void *out, const void *q, const float *scales, int64_t rows,
                          int64_t width, int32_t dtype, hipStream_t stream);

/* residual = x + add and, in 8 bits, rms(residual) * (1 + norm): qdc_residual_rmsnorm of an
 * fp32 stream with qdc_quantize_q8 in the same pass.  add NULL: residual is x and not
 * written (it may be NULL).  mask (int32 [rows], NULL: none): rows where it is 0 give zeros.
 * norm has norm_dtype; x, add, residual [rows, width] contiguous.  residual may be x. */
int32_t qdc_residual_rmsnorm_q8(float *residual, void *q, float *scales, const float *x,
                                const float *add, const void *norm, const int32_t *mask,
                                int64_t rows, int64_t width, float eps, int32_t norm_dtype,
                                hipStream_t stream);

/* y = x w^T, or with gated != 0 y = silu(x gate^T) * (x up^T): y [rows, out] ([rows, out / 2])
 * contiguous, fp32 or bf16, and of a gated product also QDC_Q8 (y_scales; out / 2 a multiple
 * of 16).  x [rows, inner], at most 2^20 - 16 rows, is fp32, bf16 (rows ld_x elements apart, a
 * multiple of 8, at most 2^26 bytes) or QDC_Q8 (x_scales; inner a multiple of 16, ld_x =
 * inner).  Sums are fp32 (whole numbers within a group of 8-bit rows), the scale applied to
 * each group's sum: q * x is summed before it and in steps of 1/16, so an fp32 or bf16 x
 * beyond 2^113 and a result beyond 2^123 may overflow where q * s * x would not; of an fp32 x
 * what lies below 2^-133 is lost.  Of 8-bit rows a weight's scale (2^127 / 3 at most, as those
 * of finite weights are) below 2^-105, a result below 2^-109 and a product of both scales
 * below 2^-126 lose bits, and such a product beyond 2^128 may overflow.
 * x_scales and y_scales are ignored where they are not used.  workspace: device memory of
 * qdc_linear_w4_workspace bytes (0 unless y is QDC_Q8, and its rows few: NULL then), 16-byte
 * aligned, the call's alone until it is done. */
int32_t qdc_linear_w4(void *y, float *y_scales, int32_t y_dtype, const void *x,
                      const float *x_scales, int32_t x_dtype, const void *packed,
                      const void *scales, int64_t rows, int64_t out, int64_t inner, int64_t group,
                      int64_t ld_x, int32_t gated, void *workspace, int64_t workspace_bytes,
                      hipStream_t stream);
/* -1 for sizes that it refuses. */
int64_t qdc_linear_w4_workspace(int64_t rows, int64_t out, int64_t inner, int64_t group,
                                int32_t gated, int32_t y_dtype);

#ifdef __cplusplus
}
#endif
#endif
