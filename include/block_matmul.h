/*
 * libblock_matmul_hip.so -- matrix product in 8-bit floating point (e4m3) with
 * a scale for each block of 128, for MI355X (gfx950).
 *
 *   out[m, n] = sum_b sa[m, b] sb[n, b] sum_{k in block b} a[m, k] b[n, k]
 *
 * a: M rows of K codes, b: N rows of K codes, `pitch` bytes between rows (a
 * multiple of 16, at least K); the memory of the last row reaches up to the
 * next multiple of 16 after K, and what lies from K on does not count.
 * Blocks are 128 numbers of a row, or (tiles != 0) 128 rows by 128 columns;
 * the scale of block b of row r (or of row of tiles r / 128) is at
 * r * row_stride + b * block_stride, in scales.  scale_type 0: float32,
 * 1: exponent + 127 in a byte (e8m0, 255 NaN), for both operands.
 *
 * out: M rows of N numbers of out_dtype (0 float32, 1 bfloat16, 2 float16),
 * dense; like all that is written it overlaps nothing else.  K is at most 2^22.
 * A block's sum and the sum over blocks are held in float32; the result is
 * rounded once.  For 16-bit results a block's products are added by the 8-bit
 * matrix instruction, which drops what lies 13 bits below the largest of each
 * eight: a result is off by at most 7 * 2^-13 of the sum of those largest ones
 * before it is rounded, however small it is itself.  Of random numbers that is
 * 1.5e-5 of the results' root mean square (measured; rounding costs 1.7e-3 in
 * bfloat16, 2.1e-4 in float16).  For float32 results they are added by the
 * 16-bit instruction, which takes 2.5 times as long and drops nothing.
 * Products of two scales are formed in float32, where they can overflow or
 * lose bits below 2^-126; for 16-bit results powers of two are exact.
 *
 * Device arrays owned by the caller; the library allocates nothing, keeps no
 * state, never synchronises and launches on `stream`.  The workspace is
 * scratch: calls that run at once need one each.  Arguments are validated
 * before any HIP call (NL2K_* codes, message from block_matmul_last_error()).
 * All results are bitwise repeatable for one set of sizes.
 */
#ifndef NL2K_BLOCK_MATMUL_H
#define NL2K_BLOCK_MATMUL_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of scratch (0: none is needed, or the call refuses these sizes). */
size_t block_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int out_dtype);

int block_matmul(const void* a, int64_t a_pitch, const void* a_scales, int64_t a_row_stride,
                 int64_t a_block_stride, int a_tiles, const void* b, int64_t b_pitch,
                 const void* b_scales, int64_t b_row_stride, int64_t b_block_stride, int b_tiles,
                 int scale_type, void* out, int out_dtype, int64_t M, int64_t N, int64_t K,
                 void* workspace, size_t workspace_bytes, hipStream_t stream);

/*
 * A layer of it: y = Q(x) Q(w)^T, dx = Q(dy) Q(w), dw = Q(dy^T) Q(x^T)^T, where
 * Q quantises x, dy and their transposes by rows and w [N, K] by tiles, as
 * block_quant.h describes.  x, dy, w, y, dx, dw: types 0, 1, 2 as above; rows of
 * x, dy and w a stride in numbers apart, written arrays dense, y and dx of x's
 * type.  w_codes, where not NULL, is w quantised already (w is not read then),
 * with its pitch, and scales of tiles at w_row_stride, w_block_stride; the
 * backward takes the transposed matrix's, [K, N].
 *
 * What a backward needs is kept by the forward in `kept`, 256-byte aligned, of
 * block_linear_kept_bytes: for dx the transposed w (unless w_codes is given),
 * for dw the transposed x.  M = 0 does nothing; dw is the caller's to clear.
 * The numbers that a product adds are at most 2^22: K for y, N where dx is
 * wanted, M where dw is.
 */
size_t block_linear_kept_bytes(int64_t M, int64_t N, int64_t K, int scale_type, int want_dx,
                               int want_dw, int have_codes);

/* Bytes of scratch, 256-byte aligned, of the forward (backward 0; x's type) or
 * the backward (1; w's type); 0 for sizes that the call refuses. */
size_t block_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int scale_type, int x_dtype,
                                    int w_dtype, int backward);

int block_linear_forward(const void* x, int x_dtype, int64_t x_stride, const void* w, int w_dtype,
                         int64_t w_stride, const void* w_codes, int64_t w_pitch,
                         const void* w_scales, int64_t w_row_stride, int64_t w_block_stride,
                         int scale_type, int want_dx, int want_dw, void* y, void* kept, int64_t M,
                         int64_t N, int64_t K, void* workspace, size_t workspace_bytes,
                         hipStream_t stream);

/* dx or dw NULL: not wanted (as the forward was told). */
int block_linear_backward(const void* dy, int x_dtype, int64_t dy_stride, const void* w_codes_t,
                          int64_t w_pitch_t, const void* w_scales_t, int64_t w_row_stride_t,
                          int64_t w_block_stride_t, int scale_type, const void* kept, void* dx,
                          void* dw, int w_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                          size_t workspace_bytes, hipStream_t stream);

const char* block_matmul_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_BLOCK_MATMUL_H */
