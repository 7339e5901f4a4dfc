// Clipped policy loss with a KL term, from logits, for MI355X (gfx950).  C-ABI
// in include/policy_loss.h, row kernels in csrc/token_rows.h.
//
// Three launches: the sum of the weights (left out where the caller gives the
// denominator, or a wave can add them up by itself), the rows, the sum of their
// terms.

#include "policy_loss.h"
#include "token_rows.h"

namespace {

using nl2k::rows::Shape;

constexpr int kSumBlocks = 64;  // most partial sums of the weights: one a lane

// Weight of a row: 0 where its label is ignored, else its mask.
struct Weights {
  const void* mask;
  int kind;
  __device__ __forceinline__ float masked(uint32_t r) const {
    if (kind == 0) return 1.f;
    if (kind == 1) return static_cast<const unsigned char*>(mask)[r] ? 1.f : 0.f;
    return static_cast<const float*>(mask)[r];
  }
  __device__ __forceinline__ float at(uint32_t r, int64_t lab, int64_t ignore) const {
    return lab == ignore ? 0.f : masked(r);
  }
  // Sum of U rows' weights, `step` apart from r on; all reads in flight together.
  template <int U>
  __device__ __forceinline__ void add(const int64_t* __restrict__ labels, uint32_t r,
                                      uint32_t step, uint32_t rows, int64_t ignore,
                                      double& s) const {
    int64_t lab[U];
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t q = min(r + u * step, rows - 1);
      lab[u] = labels[q];
      w[u] = masked(q);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u * step < rows && lab[u] != ignore) s += w[u];
  }
};

__device__ __forceinline__ double block_sum(double v, double* red) {
  v = nl2k::wave_sum(v);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

__global__ __launch_bounds__(1024) void weight_sum_kernel(const int64_t* __restrict__ labels,
                                                          Weights w, uint32_t rows, int64_t ignore,
                                                          double* __restrict__ partial) {
  __shared__ double red[16];
  double s = 0.0;
  for (uint32_t r = blockIdx.x * 4096 + threadIdx.x; r < rows; r += gridDim.x * 4096)
    w.add<4>(labels, r, 1024, rows, ignore, s);
  s = block_sum(s, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// D, given or the weights' sum.  The partial sums, of 64 bits each, are added in 32: exactly where
// they count tokens, and a row of 512 classes waits less for it than for the shuffles of a sum in
// 64.  Up to kOwnRows rows there are none and one launch less: every wave adds up all weights,
// 17.7 us a call in place of 19.6 for 16 to 512 rows of 1024 float32 (with 50257, where the call's
// time is the GPU's, 22.7 and 23.6 for 256 rows, 45.1 and 44.8 for 512).
constexpr uint32_t kOwnRows = 512;
struct Denominator {
  float given;
  const double* __restrict__ partial;
  int blocks;
  const int64_t* __restrict__ labels;
  Weights w;

  // 1 / D, or 0 where D is; the same in every lane of a wave
  __device__ __forceinline__ float inverse(uint32_t rows, int64_t ignore) const {
    float d = given;
    if (d <= 0.f) {
      const int lane = threadIdx.x & 63;
      if (blocks == 0) {
        double s = 0.0;
#pragma unroll 1
        for (uint32_t r = lane; r < rows; r += 256) w.add<4>(labels, r, 64, rows, ignore, s);
        d = nl2k::wave_sum_dpp((float)s);
      } else if (blocks == 1) {
        d = (float)partial[0];
      } else {
        d = nl2k::wave_sum_dpp(lane < blocks ? (float)partial[lane] : 0.f);
      }
    }
    return d != 0.f ? 1.f / d : 0.f;
  }
};

__global__ __launch_bounds__(1024) void loss_kernel(const float* __restrict__ terms, uint32_t rows,
                                                    Denominator den, int64_t ignore,
                                                    float* __restrict__ loss) {
  __shared__ double red[16];
  // eight pairs a thread at a time: one workgroup adds 262144 terms in 19 us
  double s = 0.0;
  const uint32_t pairs = rows / 2;
  const nl2k::f32x2* t2 = reinterpret_cast<const nl2k::f32x2*>(terms);
  for (uint32_t p = threadIdx.x; p < pairs; p += 8 * 1024) {
    nl2k::f32x2 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = t2[min(p + u * 1024, pairs - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (p + u * 1024 < pairs) s += (double)v[u][0] + (double)v[u][1];
  }
  if ((rows & 1) && threadIdx.x == 0) s += terms[rows - 1];
  const float inv = rows ? den.inverse(rows, ignore) : 0.f;
  s = block_sum(s, red);
  if (threadIdx.x == 0) loss[0] = (float)(s * inv);
}

struct PolicyOp {
  const float* __restrict__ old_logp;
  const float* __restrict__ adv;
  int64_t adv_bs, adv_ss;
  const float* __restrict__ ref;
  Weights w;
  float lo, hi, kl_coef;
  Denominator den;
  float* __restrict__ terms;
  float* __restrict__ logp;
  float* __restrict__ coef;
  float inv;  // 1 / D

  __device__ void begin(const Shape& sh) { inv = den.inverse(sh.rows, sh.ignore); }
  __device__ bool counts(const Shape& sh, uint32_t r, int64_t lab) const {
    return w.at(r, lab, sh.ignore) != 0.f;
  }
  __device__ void skip(uint32_t r, bool lead) const {
    if (!lead) return;
    terms[r] = 0.f;
    logp[r] = 0.f;
    if (coef) coef[r] = 0.f;
  }
  __device__ float finish(const Shape& sh, uint32_t r, double lp, bool lead) const {
    const uint32_t b = sh.S == sh.rows ? 0u : r / sh.S;
    const float a = adv[(int64_t)b * adv_bs + (int64_t)(r - b * sh.S) * adv_ss];
    const float weight = w.kind == 2 ? static_cast<const float*>(w.mask)[r] : 1.f;
    const float ratio = expf((float)(lp - (double)old_logp[r]));
    // selects that let a NaN through, as the products do
    const float cut = ratio < lo ? lo : ratio > hi ? hi : ratio;
    const float free_term = ratio * a, cut_term = cut * a;
    const bool held = a >= 0.f ? ratio > hi : ratio < lo;  // the clamp holds the minimum
    float term = held ? -cut_term : -free_term;
    float g = held ? 0.f : -free_term;
    if (ref) {
      const float d = (float)((double)ref[r] - lp);
      const float e = expm1f(d);
      term += kl_coef * (e - d);
      g -= kl_coef * e;
    }
    if (lead) {
      terms[r] = weight * term;
      logp[r] = (float)lp;
    }
    g *= weight * inv;
    if (lead && coef) coef[r] = g;
    return g;
  }
};

int sum_blocks(int64_t rows) {
  if (rows <= kOwnRows) return 0;
  return (int)std::min<int64_t>(kSumBlocks, nl2k::ceil_div(rows, (int64_t)4096));
}

size_t workspace_bytes_of(int64_t rows) { return kSumBlocks * 8 + (size_t)(rows + 1) / 2 * 8; }

struct Call {
  Shape sh;
  PolicyOp op;
};

// Checks what both forwards take and fills in the op.
int make_call(const char* what, const void* logits, int dtype, const int64_t* labels,
              const float* old_logp, const float* adv, int64_t adv_bs, int64_t adv_ss,
              const float* ref, const void* mask, int mask_kind, float* loss, float* logp,
              int64_t B, int64_t S, int64_t V, int64_t bs, int64_t rs, int64_t ignore,
              float temperature, float clip_low, float clip_high, float kl_coef, float denom,
              void* ws, size_t ws_bytes, Call* c) {
  int st = nl2k::rows::make_shape(B, S, V, bs, rs, ignore, temperature, dtype, &c->sh);
  if (st) return st;
  if (!loss) return nl2k::fail(NL2K_ERR_NULL, "%s: loss is required", what);
  if (mask_kind < 0 || mask_kind > 2)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: mask_kind must be 0, 1 or 2, got %d", what, mask_kind);
  if (!(clip_low >= 0.f) || !(clip_low <= 1.f) || !(clip_high >= 0.f) || !(clip_high < INFINITY))
    return nl2k::fail(NL2K_ERR_VALUE,
                      "%s: clip_low must be in [0, 1] and clip_high at least 0, got %g and %g",
                      what, (double)clip_low, (double)clip_high);
  if (!(kl_coef >= 0.f) || !(kl_coef < INFINITY))
    return nl2k::fail(NL2K_ERR_VALUE, "%s: kl_coef must be finite and at least 0, got %g", what,
                      (double)kl_coef);
  if (!(denom >= 0.f) || !(denom < INFINITY))
    return nl2k::fail(NL2K_ERR_VALUE, "%s: denom must be finite and positive, or 0 for the sum of "
                      "the weights, got %g", what, (double)denom);
  if (kl_coef > 0.f && !ref && c->sh.rows)
    return nl2k::fail(NL2K_ERR_NULL, "%s: kl_coef %g needs ref_logp", what, (double)kl_coef);
  if (c->sh.rows && (!logits || !labels || !old_logp || !adv || !logp || (mask_kind && !mask)))
    return nl2k::fail(NL2K_ERR_NULL, "%s: a required pointer is NULL", what);
  if (ws_bytes < workspace_bytes_of(c->sh.rows) || !ws)
    return nl2k::fail(NL2K_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what, ws_bytes,
                      workspace_bytes_of(c->sh.rows));
  if ((st = nl2k::rows::check_align(ws, 0, "workspace", 8))) return st;
  if ((st = nl2k::rows::check_align(logits, dtype, "logits"))) return st;
  double* partial = static_cast<double*>(ws);
  c->op = PolicyOp{old_logp, adv, adv_bs, adv_ss, kl_coef > 0.f ? ref : nullptr,
                   Weights{mask, mask_kind}, 1.f - clip_low, 1.f + clip_high, kl_coef,
                   Denominator{denom, partial, sum_blocks(c->sh.rows), labels,
                               Weights{mask, mask_kind}},
                   reinterpret_cast<float*>(partial + kSumBlocks), logp, nullptr, 0.f};
  return NL2K_SUCCESS;
}

void sum_weights(const Call& c, hipStream_t stream) {
  const Denominator& den = c.op.den;
  if (den.given > 0.f || den.blocks == 0) return;
  hipLaunchKernelGGL(weight_sum_kernel, dim3(den.blocks), dim3(1024), 0, stream, den.labels, den.w,
                     c.sh.rows, c.sh.ignore, const_cast<double*>(den.partial));
}

int sum_loss(const Call& c, float* loss, hipStream_t stream) {
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, stream, c.op.terms, c.sh.rows,
                     c.op.den, c.sh.ignore, loss);
  return nl2k::check_launch("loss_kernel");
}

}  // namespace

extern "C" size_t policy_loss_workspace_bytes(int64_t B, int64_t S) {
  if (B < 0 || S < 0 || (S && B > ((int64_t)1 << 28) / S)) return 0;
  return workspace_bytes_of(B * S);
}

extern "C" int policy_loss_forward(const void* logits, int dtype, const int64_t* labels,
                                   const float* old_logp, const float* advantages, int64_t adv_bs,
                                   int64_t adv_ss, const float* ref_logp, const void* mask,
                                   int mask_kind, float* loss, float* logp, float* stats,
                                   float* coef, int64_t B, int64_t S, int64_t V,
                                   int64_t batch_stride, int64_t row_stride, int64_t ignore_index,
                                   float temperature, float clip_low, float clip_high,
                                   float kl_coef, float denom, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  Call c;
  int st = make_call("policy_loss_forward", logits, dtype, labels, old_logp, advantages, adv_bs,
                     adv_ss, ref_logp, mask, mask_kind, loss, logp, B, S, V, batch_stride,
                     row_stride, ignore_index, temperature, clip_low, clip_high, kl_coef, denom,
                     workspace, workspace_bytes, &c);
  if (st) return st;
  if ((stats == nullptr) != (coef == nullptr))
    return nl2k::fail(NL2K_ERR_NULL, "policy_loss_forward: stats and coef come together");
  if ((st = nl2k::rows::check_align(stats, 0, "stats", 8))) return st;
  c.op.coef = coef;
  if (c.sh.rows) {
    sum_weights(c, stream);
    st = nl2k::rows::launch_forward(logits, dtype, labels, reinterpret_cast<nl2k::f32x2*>(stats),
                                    c.sh, c.op, stream);
    if (st) return st;
  }
  return sum_loss(c, loss, stream);
}

extern "C" int policy_loss_backward(const void* logits, int dtype, const int64_t* labels,
                                    const float* stats, const float* coef, const float* gout,
                                    void* dlogits, int64_t B, int64_t S, int64_t V,
                                    int64_t batch_stride, int64_t row_stride,
                                    int64_t ignore_index, float temperature, hipStream_t stream) {
  return nl2k::rows::backward("policy_loss_backward", logits, dtype, labels, stats, coef, gout,
                              dlogits, B, S, V, batch_stride, row_stride, ignore_index,
                              temperature, stream);
}

extern "C" int policy_loss_and_grad(const void* logits, int dtype, const int64_t* labels,
                                    const float* old_logp, const float* advantages, int64_t adv_bs,
                                    int64_t adv_ss, const float* ref_logp, const void* mask,
                                    int mask_kind, float* loss, float* logp, void* dlogits,
                                    int64_t B, int64_t S, int64_t V, int64_t batch_stride,
                                    int64_t row_stride, int64_t ignore_index, float temperature,
                                    float clip_low, float clip_high, float kl_coef, float denom,
                                    void* workspace, size_t workspace_bytes, hipStream_t stream) {
  Call c;
  int st = make_call("policy_loss_and_grad", logits, dtype, labels, old_logp, advantages, adv_bs,
                     adv_ss, ref_logp, mask, mask_kind, loss, logp, B, S, V, batch_stride,
                     row_stride, ignore_index, temperature, clip_low, clip_high, kl_coef, denom,
                     workspace, workspace_bytes, &c);
  if (st) return st;
  if (c.sh.rows) {
    if (!dlogits)
      return nl2k::fail(NL2K_ERR_NULL, "policy_loss_and_grad: dlogits is required");
    if ((st = nl2k::rows::check_align(dlogits, dtype, "dlogits"))) return st;
    // a dimension of one has no stride to speak of
    if (dlogits == logits &&
        ((S > 1 && row_stride != V) || (B > 1 && batch_stride != S * V)))
      return nl2k::fail(NL2K_ERR_SHAPE, "policy_loss_and_grad: in place needs dense logits");
    sum_weights(c, stream);
    st = nl2k::rows::launch_fused(logits, dtype, labels, dlogits, c.sh, c.op, stream);
    if (st) return st;
  }
  return sum_loss(c, loss, stream);
}

extern "C" const char* policy_loss_last_error(void) { return nl2k::error_slot().text; }
