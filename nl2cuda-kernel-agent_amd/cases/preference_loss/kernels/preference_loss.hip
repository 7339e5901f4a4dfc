// Preference loss of paired log ratios, from logits, for MI355X (gfx950).
// C-ABI in include/preference_loss.h, row kernels in csrc/token_rows.h.
//
// The gradient of a row needs its pair's sums over all tokens, so the logits
// are read twice: the rows' log-probabilities, a workgroup a pair that sums
// them and writes the tokens' coefficients, the last of which adds up the
// pairs' losses, and the stream that makes dlogits.

#include "preference_loss.h"
#include "token_rows.h"

namespace {

using nl2k::rows::Shape;

struct SequenceOp {
  float* __restrict__ logp;
  float* __restrict__ coef;  // zeros until the pairs are known: rows in no sequence keep them
  uint32_t* __restrict__ done;  // 0 for pair_kernel
  __device__ void begin(const Shape&) const {}
  __device__ bool counts(const Shape& sh, uint32_t, int64_t lab) const { return lab != sh.ignore; }
  __device__ void skip(uint32_t r, bool lead) const { put(r, 0.f, lead); }
  __device__ float finish(const Shape&, uint32_t r, double lp, bool lead) const {
    put(r, (float)lp, lead);
    return 0.f;
  }
  __device__ void put(uint32_t r, float lp, bool lead) const {
    if (!lead) return;
    logp[r] = lp;
    if (coef) coef[r] = 0.f;
    if (r == 0) *done = 0;
  }
};

constexpr int kPairBlock = 256;
constexpr int64_t kMostPairs = nl2k::max_blocks(kPairBlock);  // a workgroup each

__device__ __forceinline__ double block_sum(double v, double* red) {
  v = nl2k::wave_sum(v);
  __syncthreads();  // red may still be read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

// Rows of sequence i.
__device__ __forceinline__ void bounds(const int64_t* __restrict__ cu, int64_t i, const Shape& sh,
                                       uint32_t& lo, uint32_t& hi) {
  if (cu) {
    const int64_t a = min(max(cu[i], (int64_t)0), (int64_t)sh.rows);
    lo = (uint32_t)a;
    hi = (uint32_t)min(max(cu[i + 1], a), (int64_t)sh.rows);
  } else {
    lo = (uint32_t)i * sh.S;
    hi = lo + sh.S;
  }
}

__global__ void no_rows_kernel(uint32_t* done) { *done = 0; }

// `loss` counts the workgroups that are done, from 0, until the last of them has their losses' mean
// to put there.  That takes their sum in a fixed order; a launch of its own for it took 4.6 us.
__global__ __launch_bounds__(kPairBlock) void pair_kernel(
    const float* __restrict__ logp, const int64_t* __restrict__ labels,
    const float* __restrict__ ref, const int64_t* __restrict__ cu, Shape sh, uint32_t pairs,
    float beta, float eps, int average, float* __restrict__ seq_logp, float* __restrict__ coef,
    float* __restrict__ pair_loss, uint32_t* __restrict__ loss) {
  __shared__ double red[kPairBlock / 64];
  __shared__ bool last;
  double h[2];
  float share[2];
  uint32_t lo[2], hi[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t i = blockIdx.x + (uint32_t)j * pairs;
    bounds(cu, i, sh, lo[j], hi[j]);
    double s = 0.0, n = 0.0;
    for (uint32_t r = lo[j] + threadIdx.x; r < hi[j]; r += kPairBlock) {
      s += logp[r];
      n += labels[r] != sh.ignore ? 1.0 : 0.0;
    }
    s = block_sum(s, red);
    if (average) {
      n = block_sum(n, red);
      s /= fmax(n, 1.0);
      share[j] = (float)(1.0 / fmax(n, 1.0));
    } else {
      share[j] = 1.f;
    }
    if (threadIdx.x == 0) seq_logp[i] = (float)s;
    h[j] = beta * (s - (ref ? (double)ref[i] : 0.0));
  }
  const double d = h[0] - h[1];
  const double q = exp(-fabs(d));              // both sigmoids without cancellation
  const double big = 1.0 / (1.0 + q), small = q / (1.0 + q);
  const double up = d >= 0.0 ? big : small, down = d >= 0.0 ? small : big;
  if (threadIdx.x == 0) {
    const double soft = log1p(q);
    pair_loss[blockIdx.x] =
        (float)((1.0 - eps) * (soft + (d < 0.0 ? -d : 0.0)) + eps * (soft + (d > 0.0 ? d : 0.0)));
  }
  if (coef) {
    const float g = (float)(beta / (double)pairs * (eps * up - (1.0 - eps) * down));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      for (uint32_t r = lo[j] + threadIdx.x; r < hi[j]; r += kPairBlock)
        coef[r] = (j ? -g : g) * share[j];
  }
  // the thread that wrote the pair's loss releases it with its count, and has acquired those of
  // all others with the last
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(loss, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           pairs - 1;
  __syncthreads();
  if (!last) return;
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < pairs; i += kPairBlock) s += pair_loss[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *loss = __float_as_uint((float)(s / (double)pairs));
}

size_t even(size_t n) { return (n + 1) / 2 * 2; }

}  // namespace

extern "C" size_t preference_loss_workspace_bytes(int64_t B, int64_t S, int64_t pairs) {
  if (B < 0 || S < 0 || pairs < 1 || pairs > kMostPairs || (S && B > ((int64_t)1 << 28) / S))
    return 0;
  return 4 * (even((size_t)(B * S)) + even((size_t)pairs));
}

extern "C" int preference_loss_forward(const void* logits, int dtype, const int64_t* labels,
                                       const float* ref_seq, const int64_t* cu_seqlens,
                                       int64_t pairs, float* loss, float* seq_logp, float* stats,
                                       float* coef, int64_t B, int64_t S, int64_t V,
                                       int64_t batch_stride, int64_t row_stride,
                                       int64_t ignore_index, float beta, float label_smoothing,
                                       int average, void* workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
  Shape sh;
  int st = nl2k::rows::make_shape(B, S, V, batch_stride, row_stride, ignore_index, 1.f, dtype,
                                  &sh);
  if (st) return st;
  if (pairs > kMostPairs)
    return nl2k::fail(NL2K_ERR_OVERFLOW, "at most %lld pairs, got %lld", (long long)kMostPairs,
                      (long long)pairs);
  if (pairs < 1 || (!cu_seqlens && B != 2 * pairs) || (cu_seqlens && B != 1))
    return nl2k::fail(NL2K_ERR_SHAPE,
                      "need pairs >= 1 and B = 2 pairs, or B = 1 with cu_seqlens, got pairs=%lld "
                      "B=%lld", (long long)pairs, (long long)B);
  if (!(beta > -INFINITY) || !(beta < INFINITY))
    return nl2k::fail(NL2K_ERR_VALUE, "beta must be finite, got %g", (double)beta);
  if (!(label_smoothing >= 0.f) || !(label_smoothing <= 1.f))
    return nl2k::fail(NL2K_ERR_VALUE, "label_smoothing must be in [0, 1], got %g",
                      (double)label_smoothing);
  if (!loss || !seq_logp || (sh.rows && (!logits || !labels)))
    return nl2k::fail(NL2K_ERR_NULL, "preference_loss_forward: a required pointer is NULL");
  if ((stats == nullptr) != (coef == nullptr))
    return nl2k::fail(NL2K_ERR_NULL, "preference_loss_forward: stats and coef come together");
  const size_t need = preference_loss_workspace_bytes(B, S, pairs);
  if (workspace_bytes < need || !workspace)
    return nl2k::fail(NL2K_ERR_WORKSPACE,
                      "preference_loss_forward: workspace of %zu bytes, needs %zu",
                      workspace_bytes, need);
  if ((st = nl2k::rows::check_align(workspace, 0, "workspace", 8))) return st;
  if ((st = nl2k::rows::check_align(logits, dtype, "logits"))) return st;
  if ((st = nl2k::rows::check_align(stats, 0, "stats", 8))) return st;
  float* logp = static_cast<float*>(workspace);
  float* pair_loss = logp + even(sh.rows);
  uint32_t* counter = reinterpret_cast<uint32_t*>(loss);
  if (sh.rows) {
    st = nl2k::rows::launch_forward(logits, dtype, labels, reinterpret_cast<nl2k::f32x2*>(stats),
                                    sh, SequenceOp{logp, coef, counter}, stream);
    if (st) return st;
  } else {
    hipLaunchKernelGGL(no_rows_kernel, dim3(1), dim3(1), 0, stream, counter);
  }
  hipLaunchKernelGGL(pair_kernel, dim3((unsigned)pairs), dim3(kPairBlock), 0, stream, logp, labels,
                     ref_seq, cu_seqlens, sh, (uint32_t)pairs, beta, label_smoothing, average,
                     seq_logp, coef, pair_loss, counter);
  return nl2k::check_launch("pair_kernel");
}

extern "C" int preference_loss_backward(const void* logits, int dtype, const int64_t* labels,
                                        const float* stats, const float* coef, const float* gout,
                                        void* dlogits, int64_t B, int64_t S, int64_t V,
                                        int64_t batch_stride, int64_t row_stride,
                                        int64_t ignore_index, hipStream_t stream) {
  return nl2k::rows::backward("preference_loss_backward", logits, dtype, labels, stats, coef, gout,
                              dlogits, B, S, V, batch_stride, row_stride, ignore_index, 1.f,
                              stream);
}

extern "C" const char* preference_loss_last_error(void) { return nl2k::error_slot().text; }
