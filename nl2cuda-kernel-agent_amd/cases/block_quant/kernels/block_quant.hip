// Matrices in e4m3 with a scale for each block of 128, for MI355X (gfx950).
// C-ABI in include/block_quant.h, kernels in csrc/quantize.h, the arithmetic in
// csrc/e4m3.h.

#include "block_quant.h"

#include "quantize.h"

extern "C" int block_quant_rows(const void* x, int dtype, int64_t stride, void* codes,
                                int64_t pitch, void* scales, void* codes_t, int64_t pitch_t,
                                void* scales_t, int scale_type, int64_t M, int64_t K,
                                hipStream_t stream) {
  return nl2k::quant::run("block_quant_rows", x, dtype, stride, codes, pitch, scales, codes_t,
                          pitch_t, scales_t, scale_type, M, K, false, stream);
}

extern "C" int block_quant_tiles(const void* x, int dtype, int64_t stride, void* codes,
                                 int64_t pitch, void* scales, void* codes_t, int64_t pitch_t,
                                 int scale_type, int64_t M, int64_t K, hipStream_t stream) {
  return nl2k::quant::run("block_quant_tiles", x, dtype, stride, codes, pitch, scales, codes_t,
                          pitch_t, nullptr, scale_type, M, K, true, stream);
}

extern "C" const char* block_quant_last_error(void) { return nl2k::error_slot().text; }
