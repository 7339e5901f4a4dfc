/*
 * librms_norm_hip.so -- root-mean-square norm with the residual's addition,
 * forward, backward and with its output in 8 bits, for MI355X (gfx950).
 *
 *   h = x + residual, rounded to the type of the residual (h = x without one)
 *   r = 1 / sqrt(mean(h^2) + eps)
 *   y = h r weight
 *   dh' = r (g - h r mean(g h r)) + dh,   g = dy weight
 *   dweight = sum over rows of dy h r
 *
 * The norm is that of the rounded sum, which is what the residual stream goes
 * on with and what the backward reads: forward, backward and reader see the
 * same numbers.  Everything else is held in float32 and rounded once, where it
 * is stored.  dh' is the gradient of x and of the residual alike.
 *
 * x, residual, dy, h, dh: `rows` rows of D numbers, a stride in numbers
 * between rows; weight [D].  Types 0 float32, 1 bfloat16, 2 float16; the
 * residual (h, dh) of x's type or float32, the weight of any.  Written arrays
 * are dense and overlap nothing else.  Pointers are aligned to their type.
 * Up to 67108860 rows, and up to 2^31 - 16385 numbers in one.
 *
 * In 8 bits (rms_norm_quant) the output is laid out as block_quant.h's rows:
 * codes of `pitch` bytes a row, zeros up to the next multiple of 16, scales
 * [ceil(D / 128)][rows].
 *
 * Device arrays owned by the caller; the library allocates nothing, keeps no
 * state, never synchronises and launches on `stream`.  Arguments are validated
 * before any HIP call (NL2K_* codes, message from rms_norm_last_error()).
 * All results are bitwise repeatable.
 */
#ifndef NL2K_RMS_NORM_H
#define NL2K_RMS_NORM_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y, h (with a residual: required, without: NULL) and, where a backward
 * follows, rstd [rows] (NULL otherwise). */
int rms_norm_forward(const void* x, int dtype, int64_t x_stride, const void* residual,
                     int residual_dtype, int64_t residual_stride, const void* weight,
                     int weight_dtype, void* y, void* h, float* rstd, int64_t rows, int64_t D,
                     float eps, hipStream_t stream);

/* The same with y as codes and scales. */
int rms_norm_quant(const void* x, int dtype, int64_t x_stride, const void* residual,
                   int residual_dtype, int64_t residual_stride, const void* weight,
                   int weight_dtype, void* codes, int64_t pitch, void* scales, int scale_type,
                   void* h, int64_t rows, int64_t D, float eps, hipStream_t stream);

/* Bytes of scratch for dweight; 0 for sizes that the call refuses. */
size_t rms_norm_backward_workspace_bytes(int64_t rows, int64_t D);

/* dx of dy's type; dresidual of h's type, NULL where the types agree (dx is
 * it then) or it is not wanted.  dh NULL: h has no gradient of its own.
 * dweight NULL: not wanted, and no workspace is needed. */
int rms_norm_backward(const void* dy, int dtype, int64_t dy_stride, const void* h, int h_dtype,
                      int64_t h_stride, const void* dh, int64_t dh_stride, const void* weight,
                      int weight_dtype, const float* rstd, void* dx, void* dresidual,
                      void* dweight, int64_t rows, int64_t D, void* workspace,
                      size_t workspace_bytes, hipStream_t stream);

const char* rms_norm_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_RMS_NORM_H */
