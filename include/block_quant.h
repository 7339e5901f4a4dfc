/*
 * libblock_quant_hip.so -- matrices in 8-bit floating point (e4m3) with a
 * scale for each block of 128 numbers, for MI355X (gfx950).
 *
 *   rows:   a block is 128 numbers of a row (the last one what is left)
 *   tiles:  a block is 128 rows by 128 columns (the last ones what is left)
 *   s = max(a / 448, 2^-126), a the block's largest magnitude, in float32
 *       (scale_type 0); or the least power of two that is no smaller, kept as
 *       exponent + 127 in a byte (scale_type 1, "e8m0")
 *   code = e4m3(x * fl(1 / s)), to nearest even
 *
 * x: M rows of K numbers of float32, bfloat16 or float16 (dtype 0, 1, 2),
 * aligned to a number, rows `stride` numbers apart.  codes: M rows of K bytes,
 * `pitch` apart, a multiple of 16 and at least K; the bytes from K up to the
 * next multiple of 16 are written as zeros.  Scales of rows: [ceil(K / 128)][M],
 * blocks first, as the product reads them; of tiles: [ceil(M / 128)][ceil(K / 128)].
 *
 * codes_t, where not NULL, takes the transposed matrix, K rows of M bytes,
 * pitch_t apart.  For rows its blocks run along M, with scales of their own:
 * scales_t [ceil(M / 128)][K].  For tiles it holds the same codes, under the
 * same scales (scales_t is not used).  x is read once either way.
 *
 * A NaN stays in its own code.  An infinity makes its scale infinite (e8m0:
 * NaN), and with it what the whole block stands for.
 *
 * Device arrays owned by the caller; the library allocates nothing, keeps no
 * state, never synchronises and launches on `stream`.  Arguments are validated
 * before any HIP call (NL2K_* codes, message from block_quant_last_error()).
 * All results are bitwise repeatable.
 */
#ifndef NL2K_BLOCK_QUANT_H
#define NL2K_BLOCK_QUANT_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "nl2k_status.h"

#ifdef __cplusplus
extern "C" {
#endif

int block_quant_rows(const void* x, int dtype, int64_t stride, void* codes, int64_t pitch,
                     void* scales, void* codes_t, int64_t pitch_t, void* scales_t, int scale_type,
                     int64_t M, int64_t K, hipStream_t stream);

int block_quant_tiles(const void* x, int dtype, int64_t stride, void* codes, int64_t pitch,
                      void* scales, void* codes_t, int64_t pitch_t, int scale_type, int64_t M,
                      int64_t K, hipStream_t stream);

const char* block_quant_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NL2K_BLOCK_QUANT_H */
