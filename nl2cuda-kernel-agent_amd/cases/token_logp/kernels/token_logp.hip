// Log-probabilities of given tokens, forward and backward, for MI355X
// (gfx950).  C-ABI in include/token_logp.h, kernels in csrc/token_rows.h.

#include "token_logp.h"
#include "token_rows.h"

namespace {

using nl2k::rows::Shape;

// The log-probability itself.
struct LogpOp {
  float* logp;
  __device__ void begin(const Shape&) const {}
  __device__ bool counts(const Shape& sh, uint32_t, int64_t lab) const { return lab != sh.ignore; }
  __device__ void skip(uint32_t r, bool lead) const {
    if (lead) logp[r] = 0.f;
  }
  __device__ float finish(const Shape&, uint32_t r, double lp, bool lead) const {
    if (lead) logp[r] = (float)lp;
    return 0.f;
  }
};

}  // namespace

extern "C" int token_logp_forward(const void* logits, int dtype, const int64_t* labels,
                                  float* logp, float* stats, int64_t B, int64_t S, int64_t V,
                                  int64_t batch_stride, int64_t row_stride, int64_t ignore_index,
                                  float temperature, hipStream_t stream) {
  Shape sh;
  int st = nl2k::rows::make_shape(B, S, V, batch_stride, row_stride, ignore_index, temperature,
                                  dtype, &sh);
  if (st) return st;
  if (sh.rows == 0) return nl2k::succeed();
  if (!logits || !labels || !logp)
    return nl2k::fail(NL2K_ERR_NULL, "token_logp_forward: logits, labels and logp are required");
  if ((st = nl2k::rows::check_align(logits, dtype, "logits"))) return st;
  if ((st = nl2k::rows::check_align(stats, nl2k::rows::kF32, "stats", 8))) return st;
  return nl2k::rows::launch_forward(logits, dtype, labels, reinterpret_cast<nl2k::f32x2*>(stats),
                                    sh, LogpOp{logp}, stream);
}

extern "C" int token_logp_backward(const void* logits, int dtype, const int64_t* labels,
                                   const float* stats, const float* dlogp, const float* gout,
                                   void* dlogits, int64_t B, int64_t S, int64_t V,
                                   int64_t batch_stride, int64_t row_stride, int64_t ignore_index,
                                   float temperature, hipStream_t stream) {
  return nl2k::rows::backward("token_logp_backward", logits, dtype, labels, stats, dlogp, gout,
                              dlogits, B, S, V, batch_stride, row_stride, ignore_index,
                              temperature, stream);
}

extern "C" const char* token_logp_last_error(void) { return nl2k::error_slot().text; }
