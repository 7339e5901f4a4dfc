// Rows of logits and the tokens given for them: the kernels that the token
// log-probabilities, the policy loss and the preference loss share.
//
//   m = max_v x[v],  S = sum_v exp((x[v] - m) / tau)
//   logp = (x[label] - m) / tau - log S
//   d/dx[v] (g logp) = g / tau ([v == label] - exp((x[v] - m) / tau) / S)
//
// A row is read in windows of 16 bytes from its own start, at any alignment;
// the last window of a row that is no multiple of them reaches back over the
// one before, so nothing outside the row is read or written.  Rows are found
// by two strides (batch, position), so a next-token view logits[:, :-1] is
// read where it lies.
//
// x - m is formed before it is scaled: rows of a type's lowest value stay
// finite (their softmax is uniform), and a common offset of the logits costs
// no bits.  Maxima and sums are held in 32 bits, a log-probability in 64 until
// it is stored or has had another taken from it, in 32 then; only dlogits is
// rounded, once, to the type of the logits.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"

namespace nl2k {
namespace rows {

// Types of logits, as the C entries take them.
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

struct bf16_t {};
struct f16_t {};

template <class T>
struct Elem;
template <>
struct Elem<float> {
  using type = float;
  static constexpr int E = 4;
};
template <>
struct Elem<bf16_t> {
  using type = unsigned short;
  static constexpr int E = 8;
};
template <>
struct Elem<f16_t> {
  using type = unsigned short;
  static constexpr int E = 8;
};

// 16 bytes at any alignment.
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <class T>
__device__ __forceinline__ void unpack(u32x4 w, float (&x)[Elem<T>::E]) {
  if constexpr (Elem<T>::E == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = w[i];  // a copy: the cast of a vector's element takes its first one
      x[i] = __builtin_bit_cast(float, q);
    }
  } else if constexpr (__is_same(T, bf16_t)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __builtin_bit_cast(float, w[i] << 16);
      x[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = w[i];
      const f16x2 h = __builtin_bit_cast(f16x2, q);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
}

// Round to nearest even.
template <class T>
__device__ __forceinline__ u32x4 pack(const float (&x)[Elem<T>::E]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Elem<T>::E == 4) {
      w[i] = __builtin_bit_cast(uint32_t, x[i]);
    } else if constexpr (__is_same(T, bf16_t)) {
      bf16x2 h;
      h[0] = (__bf16)x[2 * i];
      h[1] = (__bf16)x[2 * i + 1];
      w[i] = __builtin_bit_cast(uint32_t, h);
    } else {
      f16x2 h;
      h[0] = (_Float16)x[2 * i];
      h[1] = (_Float16)x[2 * i + 1];
      w[i] = __builtin_bit_cast(uint32_t, h);
    }
  }
  return w;
}

template <class T>
__device__ __forceinline__ float load_one(const typename Elem<T>::type* p) {
  if constexpr (Elem<T>::E == 4)
    return *p;
  else if constexpr (__is_same(T, bf16_t))
    return __builtin_bit_cast(float, (uint32_t)*p << 16);
  else
    return (float)__builtin_bit_cast(_Float16, *p);
}

template <class T>
__device__ __forceinline__ typename Elem<T>::type round_one(float x) {
  if constexpr (Elem<T>::E == 4)
    return x;
  else if constexpr (__is_same(T, bf16_t))
    return __builtin_bit_cast(unsigned short, (__bf16)x);
  else
    return __builtin_bit_cast(unsigned short, (_Float16)x);
}

// Logits of `rows` tokens: row r starts at element (r / S) * bs + (r % S) * rs.
struct Shape {
  uint32_t rows, S;
  int32_t V;
  int64_t bs, rs;
  int64_t ignore;   // label of rows that count for nothing
  float inv_tau;
  double inv_tau64;
  // how a launch goes about it, see `Caches`
  bool once = false;        // rows are read past the caches
  bool last_first = false;  // rows in falling order

  __device__ __forceinline__ int64_t at(uint32_t r) const {
    const uint32_t b = S == rows ? 0u : r / S;
    return (int64_t)b * bs + (int64_t)(r - b * S) * rs;
  }
};

// Column of a label, or -1 outside [0, V): such a row's answers are NaN.
__device__ __forceinline__ int label_col(int64_t lab, int32_t V) {
  return lab >= 0 && lab < V ? (int)lab : -1;
}

// What exponents are taken from: the maximum, or 0 for a row of -inf, whose sum is then 0 and
// whose logp is -inf - -inf, NaN, as the definition has it.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A maximum m and the sum s of exponentials from it, over part of a row.
struct Stat {
  float m, s;
};

// Statistics of all TPR threads of a row; every thread gets the same bits.
// k = log2(e) / tau.  red: 2 * TPR / 64 floats, unused with one wave.
template <int TPR>
__device__ __forceinline__ Stat row_stat(Stat t, float k, float* red) {
  const float mw = wave_max_dpp(t.m);
  // a thread whose share of the row is -inf, or empty, has s = 0 (or NaN)
  float sw = wave_sum_dpp(t.m == mw ? t.s : t.s * exp2_of((t.m - finite_max(mw)) * k));
  if constexpr (TPR == 64) {
    return Stat{mw, sw};
  } else {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = mw;
      red[2 * wave + 1] = sw;
    }
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, red[2 * i]);
    const float base = finite_max(m);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float mi = red[2 * i], si = red[2 * i + 1];
      s += mi == m ? si : si * exp2_of((mi - base) * k);
    }
    return Stat{m, s};
  }
}

// (x[label] - m) / tau - log S, NaN for a label outside the row.  In 64 bits, the logarithm's
// whole part apart: around 10, where logp is a row of 50257's, 32 bits round to 5e-7, which the
// losses' differences of two log-probabilities would keep.
__device__ __forceinline__ double logp_of(Stat st, float xl, int col, double inv_tau) {
  const double log2_s = (double)__builtin_amdgcn_frexp_expf(st.s) +
                        (double)__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(st.s));
  const double v = ((double)xl - (double)finite_max(st.m)) * inv_tau - log2_s * kLn2;
  return col >= 0 ? v : (double)NAN;
}

// Threads of a workgroup that share a row, TPR = 64, 256, 512 or 1024; a wave a
// row puts four rows into a workgroup.
template <int TPR>
constexpr int block_of() {
  return TPR < 256 ? 256 : TPR;
}

// The row of this thread, and whether there is one.
__device__ __forceinline__ uint32_t my_block(const Shape& sh) {
  return sh.last_first ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_of(uint32_t block) {
  if constexpr (TPR == 64)
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(block * 4 + (threadIdx.x >> 6)));
  else
    return block;
}
template <int TPR>
__device__ __forceinline__ int my_lane() {
  return TPR == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
}

// 16 bytes, past the caches or through them.  (A branch around the two would not do: the compiler
// makes one of them, through the caches.)
template <bool kPast>
__device__ __forceinline__ u32x4 load16(const void* p) {
  if constexpr (kPast)
    return __builtin_nontemporal_load(static_cast<const u32x4_u*>(p));
  else
    return *static_cast<const u32x4_u*>(p);
}
template <bool kPast>
__device__ __forceinline__ void store16(void* p, u32x4 w) {
  if constexpr (kPast)
    __builtin_nontemporal_store(w, static_cast<u32x4_u*>(p));
  else
    *static_cast<u32x4_u*>(p) = w;
}

// Statistics of a row of at least one window, read in one pass with a running
// maximum, U windows in flight a thread.
template <class T, int TPR, int U, bool kOnce = false>
__device__ __forceinline__ Stat scan_row(const typename Elem<T>::type* x, int32_t V, float k,
                                         int lane) {
  constexpr int E = Elem<T>::E;
  const int n = (V + E - 1) / E;
  Stat st{-INFINITY, 0.f};
  for (int base = 0; base < n; base += TPR * U) {
    // a wave of its own row passes over windows that no lane has
    auto none = [&](int u) { return TPR == 64 && u && base + u * TPR >= n; };
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (none(u)) break;
      const int i = min(base + lane + u * TPR, n - 1);
      w[u] = load16<kOnce>(x + min(i * E, V - E));
    }
    float v[U][E];
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (none(u)) break;
      const int i = base + lane + u * TPR;
      unpack<T>(w[u], v[u]);
      if (base + (u + 1) * TPR >= n) {  // may hold the row's last window, or none
        const int skip = i < n ? max(i * E - (V - E), 0) : E;
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] = e < skip ? -INFINITY : v[u][e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) cm = fmaxf(cm, v[u][e]);
    }
    const float nm = fmaxf(st.m, cm);
    const float b = finite_max(nm);
    float cs = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (none(u)) break;
#pragma unroll
      for (int e = 0; e < E; ++e) cs += exp2_of((v[u][e] - b) * k);
    }
    st.s = st.s * exp2_of((st.m - b) * k) + cs;
    st.m = nm;
  }
  return st;
}

// Statistics of a row of fewer elements than a window.
template <class T, int TPR>
__device__ __forceinline__ Stat scan_short(const typename Elem<T>::type* x, int32_t V, float k,
                                           int lane) {
  const float v = lane < V ? load_one<T>(x + lane) : -INFINITY;
  return Stat{v, exp2_of((v - finite_max(v)) * k)};
}

// g ([c == label] - p) of window i in place of x.  coef = g / tau, scale = coef / S.
template <class T>
__device__ __forceinline__ u32x4 gradient(u32x4 w, int c0, int col, float m, float k, float coef,
                                          float scale) {
  constexpr int E = Elem<T>::E;
  float v[E];
  unpack<T>(w, v);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = -scale * exp2_of((v[e] - m) * k);
  const int off = col - c0;
  if ((unsigned)off < (unsigned)E) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += e == off ? coef : 0.f;
  }
  return pack<T>(v);
}

template <class T, bool kPast>
__device__ __forceinline__ void store_window(typename Elem<T>::type* __restrict__ d, int i, int n,
                                             int32_t V, u32x4 w) {
  constexpr int E = Elem<T>::E;
  const int c0 = i * E;
  if (c0 <= V - E) {
    store16<kPast>(d + c0, w);
  } else if (i < n) {  // what the window before has is left to it: d may be the logits
    const int skip = c0 - (V - E);
    typename Elem<T>::type* p = d + (V - E);
    const auto a = __builtin_bit_cast(
        typename Elem<T>::type __attribute__((ext_vector_type(Elem<T>::E))), w);
#pragma unroll
    for (int e = 1; e < E; ++e)
      if (e >= skip) p[e] = a[e];
  }
}

// Zeros over a row of the gradient.
template <class T, int TPR, bool kPast>
__device__ __forceinline__ void zero_row(typename Elem<T>::type* __restrict__ d, int32_t V,
                                         int lane) {
  constexpr int E = Elem<T>::E;
  const int n = V / E;
  for (int i = lane; i < n; i += TPR)
    store16<kPast>(d + i * E, u32x4{0u, 0u, 0u, 0u});
  if (lane < V - n * E) d[n * E + lane] = 0;
}

// What a row's statistics are turned into.  Ops of the kernels below have
//   void begin(shape)               what all rows need, read beside the row's label
//   bool counts(shape, r, label)    whether the row counts (read before the row is)
//   float finish(shape, r, logp, lead)   called by every thread with the row's logp, in
//                                   64 bits; the coefficient of its gradient.  The thread
//                                   with `lead` writes what is per token.
//   void skip(r, lead)              for rows that do not count

// Forward: the statistics (m, S) of every row, for a backward, and the op's answers.  Bound by
// memory: 50 us for 2432 rows of 50257 bfloat16, 109 for 3431 of float32 (4.9 and 6.3 TB/s).
template <class T, int TPR, int U, class Op>
__global__ __launch_bounds__(block_of<TPR>()) void forward_kernel(
    const typename Elem<T>::type* __restrict__ logits, const int64_t* __restrict__ labels,
    f32x2* __restrict__ stats, Shape sh, Op op) {
  __shared__ float red[2 * block_of<TPR>() / 64];
  const uint32_t r = row_of<TPR>(my_block(sh));
  const int lane = my_lane<TPR>();
  if (r >= sh.rows) return;
  const int64_t lab = labels[r];
  op.begin(sh);
  const bool lead = lane == 0;
  if (!op.counts(sh, r, lab)) {
    op.skip(r, lead);
    if (lead && stats) stats[r] = f32x2{0.f, 1.f};
    return;
  }
  const auto* x = logits + sh.at(r);
  const int col = label_col(lab, sh.V);
  const float xl = load_one<T>(x + max(col, 0));
  const float k = kLog2e * sh.inv_tau;
  const Stat t = sh.V < Elem<T>::E ? scan_short<T, TPR>(x, sh.V, k, lane)
                 : sh.once         ? scan_row<T, TPR, U, true>(x, sh.V, k, lane)
                                   : scan_row<T, TPR, U>(x, sh.V, k, lane);
  const Stat st = row_stat<TPR>(t, k, red);
  op.finish(sh, r, logp_of(st, xl, col, sh.inv_tau64), lead);
  if (lead && stats) stats[r] = f32x2{st.m, st.s};
}

// What of a gradient's kernel goes past the caches: nothing, its stores, its loads too.
enum Past { kNone, kStores, kBoth };

// Backward: a pure stream (238 us for 3447 rows of 50257 float32, 5.8 TB/s), TPR
// threads and U windows each a workgroup's share of a row.  coef [rows] is the
// gradient of logp; gout, where given, one number that scales it.
template <class T, int TPR, int U, Past kPast>
__global__ __launch_bounds__(block_of<TPR>()) void backward_kernel(
    const typename Elem<T>::type* __restrict__ logits, const int64_t* __restrict__ labels,
    const f32x2* __restrict__ stats, const float* __restrict__ coef,
    const float* __restrict__ gout, typename Elem<T>::type* __restrict__ dlogits, Shape sh,
    uint32_t segs) {
  constexpr int E = Elem<T>::E;
  uint32_t r = row_of<TPR>(my_block(sh)), seg = 0;
  if constexpr (TPR != 64) {
    const uint32_t block = r;
    r = block / segs;
    seg = block - r * segs;
  }
  if (r >= sh.rows) return;
  const int lane = my_lane<TPR>();
  const int64_t lab = labels[r];
  // an ignored row, or one without a gradient, gets zeros whatever its logits and gout hold
  const float c = lab == sh.ignore ? 0.f : coef[r];
  const float g = c == 0.f ? 0.f : c * (gout ? gout[0] : 1.f) * sh.inv_tau;
  const f32x2 st = stats[r];
  const int V = sh.V, n = (V + E - 1) / E;
  auto* d = dlogits + (int64_t)r * V;
  const int base = (int)seg * TPR * U, first = base + lane;
  if (g == 0.f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = first + u * TPR;
      if (V >= E && base + u * TPR < n)
        store_window<T, kPast != kNone>(d, i, n, V, u32x4{0u, 0u, 0u, 0u});
    }
    if (V < E && lane < V) d[lane] = 0;
    return;
  }
  const auto* x = logits + sh.at(r);
  const int col = label_col(lab, V);
  const float k = kLog2e * sh.inv_tau;
  const float m = finite_max(st[0]);
  const float coef_t = col >= 0 ? g : NAN;
  const float scale = coef_t / st[1];
  if (V < E) {
    if (lane < V)
      d[lane] = round_one<T>((lane == col ? coef_t : 0.f) -
                             scale * exp2_of((load_one<T>(x + lane) - m) * k));
    return;
  }
  u32x4 w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = min(first + u * TPR, n - 1);
    if (base + u * TPR < n) w[u] = load16<kPast == kBoth>(x + min(i * E, V - E));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (base + u * TPR >= n) break;
    const int i = first + u * TPR;
    const u32x4 y = gradient<T>(w[u], min(i * E, V - E), col, m, k, coef_t, scale);
    store_window<T, kPast != kNone>(d, i, n, V, y);
  }
}

// Loss terms and gradient in one pass: the row stays in registers, K windows a
// thread, between its statistics and its gradient.  4096 rows of 128256 bfloat16:
// 407 us a call, 5.2 TB/s; apart, the two passes read the logits twice.
template <class T, int TPR, int K, Past kPast, class Op>
__global__ __launch_bounds__(block_of<TPR>()) void fused_kernel(
    const typename Elem<T>::type* logits, const int64_t* __restrict__ labels,
    typename Elem<T>::type* dlogits, Shape sh, Op op) {
  constexpr int E = Elem<T>::E;
  __shared__ float red[2 * block_of<TPR>() / 64];
  const uint32_t r = row_of<TPR>(my_block(sh));
  const int lane = my_lane<TPR>();
  if (r >= sh.rows) return;
  const int64_t lab = labels[r];
  op.begin(sh);
  const bool lead = lane == 0;
  const int V = sh.V, n = (V + E - 1) / E;
  if (!op.counts(sh, r, lab)) {
    op.skip(r, lead);
    zero_row<T, TPR, kPast != kNone>(dlogits + (int64_t)r * V, V, lane);
    return;
  }
  const auto* x = logits + sh.at(r);
  const int col = label_col(lab, V);
  const float k = kLog2e * sh.inv_tau;
  const float xl = load_one<T>(x + max(col, 0));
  u32x4 w[K];
#pragma unroll
  for (int u = 0; u < K; ++u) {
    const int i = min(lane + u * TPR, n - 1);
    w[u] = load16<kPast == kBoth>(x + min(i * E, V - E));
  }
  Stat t{-INFINITY, 0.f};
#pragma unroll
  for (int u = 0; u < K; ++u) {
    if (u * TPR < n) {
      float v[E];
      unpack<T>(w[u], v);
      // the last window repeats, it does not raise the maximum; windows past it are copies
#pragma unroll
      for (int e = 0; e < E; ++e) t.m = fmaxf(t.m, v[e]);
    }
  }
  const float b = finite_max(t.m);
#pragma unroll
  for (int u = 0; u < K; ++u) {
    if (u * TPR < n) {
      float v[E];
      unpack<T>(w[u], v);
      const int i = lane + u * TPR;
      if ((u + 1) * TPR >= n) {
        const int skip = i < n ? max(i * E - (V - E), 0) : E;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < skip ? -INFINITY : v[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) t.s += exp2_of((v[e] - b) * k);
    }
  }
  // d may be the logits: the label's has to be here, not on its way, before another wave of
  // this row passes row_stat's barriers and overwrites it
  asm volatile("" : : "v"(xl));
  const Stat st = row_stat<TPR>(t, k, red);
  const float g = op.finish(sh, r, logp_of(st, xl, col, sh.inv_tau64), lead) * sh.inv_tau;
  const float m = finite_max(st.m);
  const float scale = g / st.s;
  auto* d = dlogits + (int64_t)r * V;
#pragma unroll
  for (int u = 0; u < K; ++u) {
    if (u * TPR < n) {
      const int i = lane + u * TPR;
      const u32x4 y = gradient<T>(w[u], min(i * E, V - E), col, m, k, g, scale);
      store_window<T, kPast != kNone>(d, i, n, V, y);
    }
  }
}

// The same for rows that no workgroup's registers hold, and for those below a
// window: read twice, the second time from the caches.
template <class T, int TPR, int U, bool kPast, class Op>
__global__ __launch_bounds__(block_of<TPR>()) void fused_long_kernel(
    const typename Elem<T>::type* logits, const int64_t* __restrict__ labels,
    typename Elem<T>::type* dlogits, Shape sh, Op op) {
  constexpr int E = Elem<T>::E;
  __shared__ float red[2 * block_of<TPR>() / 64];
  const uint32_t r = row_of<TPR>(my_block(sh));
  const int lane = my_lane<TPR>();
  if (r >= sh.rows) return;
  const int64_t lab = labels[r];
  op.begin(sh);
  const bool lead = lane == 0;
  const int V = sh.V, n = (V + E - 1) / E;
  auto* d = dlogits + (int64_t)r * V;
  if (!op.counts(sh, r, lab)) {
    op.skip(r, lead);
    zero_row<T, TPR, kPast>(d, V, lane);
    return;
  }
  const auto* x = logits + sh.at(r);
  const int col = label_col(lab, V);
  const float k = kLog2e * sh.inv_tau;
  const float xl = load_one<T>(x + max(col, 0));
  const Stat t = V >= E ? scan_row<T, TPR, U>(x, V, k, lane) : scan_short<T, TPR>(x, V, k, lane);
  // d may be the logits: the label's has to be here, not on its way, before another wave of
  // this row passes row_stat's barriers and overwrites it
  asm volatile("" : : "v"(xl));
  const Stat st = row_stat<TPR>(t, k, red);
  const float g = op.finish(sh, r, logp_of(st, xl, col, sh.inv_tau64), lead) * sh.inv_tau;
  const float m = finite_max(st.m);
  const float scale = g / st.s;
  if (V < E) {
    if (lane < V)
      d[lane] = round_one<T>((lane == col ? g : 0.f) -
                             scale * exp2_of((load_one<T>(x + lane) - m) * k));
    return;
  }
  for (int base = 0; base < n; base += TPR * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(base + lane + u * TPR, n - 1);
      w[u] = *reinterpret_cast<const u32x4_u*>(x + min(i * E, V - E));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + lane + u * TPR;
      const u32x4 y = gradient<T>(w[u], min(i * E, V - E), col, m, k, g, scale);
      store_window<T, kPast>(d, i, n, V, y);
    }
  }
}

// -------------------------------------------------------------- host side
// Calls f(Elem tag) for a type code.
template <class F>
inline int with_type(int dtype, F f) {
  switch (dtype) {
    case kF32: return f(float{});
    case kBF16: return f(bf16_t{});
    case kF16: return f(f16_t{});
  }
  return fail(NL2K_ERR_VALUE, "dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d",
              dtype);
}

// Sizes, strides and scalars of a call into `sh`.
inline int make_shape(int64_t B, int64_t S, int64_t V, int64_t bs, int64_t rs, int64_t ignore,
                      float temperature, int dtype, Shape* sh) {
  if (dtype < kF32 || dtype > kF16)
    return fail(NL2K_ERR_VALUE, "dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d",
                dtype);
  if (B < 0 || S < 0 || V < 1)
    return fail(NL2K_ERR_SHAPE, "need B >= 0, S >= 0 and V >= 1, got B=%lld S=%lld V=%lld",
                (long long)B, (long long)S, (long long)V);
  if (bs < 0 || rs < 0) return fail(NL2K_ERR_SHAPE, "strides of the logits must not be negative");
  if (!(temperature >= 1e-30f) || !(temperature <= 1e30f))
    return fail(NL2K_ERR_VALUE, "temperature must be from 1e-30 to 1e30, got %g",
                (double)temperature);
  // rows are counted, and a row's columns addressed, in 32 bits
  if (V > (int64_t)1 << 28 || (S && B > ((int64_t)1 << 28) / S))
    return fail(NL2K_ERR_OVERFLOW, "at most 2^28 tokens and 2^28 columns, got B=%lld S=%lld V=%lld",
                (long long)B, (long long)S, (long long)V);
  *sh = Shape{(uint32_t)(B * S), (uint32_t)(B == 1 ? B * S : S), (int32_t)V, bs, rs, ignore,
              1.f / temperature, 1.0 / (double)temperature};
  if (B == 1) sh->bs = 0;
  return NL2K_SUCCESS;
}

inline int check_align(const void* p, int dtype, const char* what, uintptr_t a = 0) {
  if (!a) a = dtype == kF32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p) % a)
    return fail(NL2K_ERR_ALIGN, "%s must be aligned to %d bytes", what, (int)a);
  return NL2K_SUCCESS;
}

// How a launch uses the caches, 32 MiB of L2 and 256 behind it, by the logits' bytes.  Times in
// us, of 8 sequences of 50257 float32 and 32000 bfloat16, through the caches first.
struct Caches {
  static constexpr int64_t kMiB = 1 << 20;
  // Rows are read past them above 160 MiB by what reads them once or for the last time: a forward
  // alone, 38 and 35 at 192, 91 and 82 at 512, but 23 and 25 at 128, found there since the call
  // before; a pass for loss and gradient, 86 and 81 at 192, 207 and 196 at 512, but 52 and 59 at
  // 128; a backward, with its forward 290 and 276 at 512, but 70 and 75 at 128.
  static constexpr int64_t kOnce = 160 * kMiB;
  // A forward whose backward comes reads past them only above 384, where that would find too
  // little: 177 and 183 for both at 320, 296 and 288 at 512.  Up to there the backward begins with
  // the rows read last: 222 and 215 at 384.
  static constexpr int64_t kTwice = 384 * kMiB;
  // Gradients above 64 MiB are written past them, where they would put the logits out: 128 and
  // 103 for a forward and backward of 192, 59 and 52 for both in one pass of 128.  Smaller ones
  // are left there for who reads them.
  static constexpr int64_t kGradient = 64 * kMiB;
};

template <class T>
inline int64_t bytes_of(const Shape& sh) {
  return (int64_t)sh.rows * sh.V * (int64_t)sizeof(typename Elem<T>::type);
}

// f(std::integral_constant of what goes past the caches) for a kernel that writes a gradient.
template <class T, class F>
inline void with_past(const Shape& sh, F f) {
  const int64_t bytes = bytes_of<T>(sh);
  if (bytes > Caches::kOnce)
    f(std::integral_constant<Past, kBoth>{});
  else if (bytes > Caches::kGradient)
    f(std::integral_constant<Past, kStores>{});
  else
    f(std::integral_constant<Past, kNone>{});
}

// Workgroups of a launch over all rows.
template <int TPR>
inline int row_grid(const Shape& sh, int64_t segs, unsigned* grid) {
  const int64_t n = TPR == 64 ? ceil_div(sh.rows, 4) : sh.rows * segs;
  if (n > max_blocks(block_of<TPR>()))
    return fail(NL2K_ERR_OVERFLOW, "%u rows of %d columns need more workgroups than a launch has",
                sh.rows, sh.V);
  *grid = (unsigned)n;
  return NL2K_SUCCESS;
}

template <class T, int TPR, int U, class Op>
inline int launch_forward_at(const void* logits, const int64_t* labels, f32x2* stats,
                             const Shape& sh, const Op& op, hipStream_t s) {
  unsigned grid;
  if (const int st = row_grid<TPR>(sh, 1, &grid)) return st;
  hipLaunchKernelGGL((forward_kernel<T, TPR, U, Op>), dim3(grid), dim3(block_of<TPR>()), 0, s,
                     static_cast<const typename Elem<T>::type*>(logits), labels, stats, sh, op);
  return check_launch("forward_kernel");
}

template <class Op>
inline int launch_forward(const void* logits, int dtype, const int64_t* labels, f32x2* stats,
                          Shape sh, const Op& op, hipStream_t s) {
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int n = (sh.V + Elem<T>::E - 1) / Elem<T>::E;
    sh.once = bytes_of<T>(sh) > (stats ? Caches::kTwice : Caches::kOnce);
    // a wave a row, no more windows at a time than there are: 65536 rows of 512 bfloat16 took
    // 37 us with four in place of one, whose exponentials were for nothing, against 21
    if (n <= 64) return launch_forward_at<T, 64, 1>(logits, labels, stats, sh, op, s);
    if (n <= 128) return launch_forward_at<T, 64, 2>(logits, labels, stats, sh, op, s);
    if (n <= 256) return launch_forward_at<T, 64, 4>(logits, labels, stats, sh, op, s);
    if (n <= 512) return launch_forward_at<T, 64, 8>(logits, labels, stats, sh, op, s);
    // few long rows: more lanes for each
    if (sh.rows >= 1024 || n <= 1024)
      return launch_forward_at<T, 256, 4>(logits, labels, stats, sh, op, s);
    return launch_forward_at<T, 512, 4>(logits, labels, stats, sh, op, s);
  });
}

template <class T, int TPR, int U>
inline int launch_backward_at(const void* logits, const int64_t* labels, const f32x2* stats,
                              const float* coef, const float* gout, void* dlogits, const Shape& sh,
                              int64_t segs, hipStream_t s) {
  unsigned grid;
  if (const int st = row_grid<TPR>(sh, segs, &grid)) return st;
  with_past<T>(sh, [&](auto past) {
    hipLaunchKernelGGL((backward_kernel<T, TPR, U, past()>), dim3(grid), dim3(block_of<TPR>()), 0,
                       s, static_cast<const typename Elem<T>::type*>(logits), labels, stats, coef,
                       gout, static_cast<typename Elem<T>::type*>(dlogits), sh, (uint32_t)segs);
  });
  return check_launch("backward_kernel");
}

inline int launch_backward(const void* logits, int dtype, const int64_t* labels,
                           const f32x2* stats, const float* coef, const float* gout,
                           void* dlogits, Shape sh, hipStream_t s) {
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int n = (sh.V + Elem<T>::E - 1) / Elem<T>::E;
    sh.last_first = bytes_of<T>(sh) <= Caches::kTwice;
    if (n <= 128)
      return launch_backward_at<T, 64, 2>(logits, labels, stats, coef, gout, dlogits, sh, 1, s);
    if (n <= 256)
      return launch_backward_at<T, 64, 4>(logits, labels, stats, coef, gout, dlogits, sh, 1, s);
    if (n <= 512)
      return launch_backward_at<T, 64, 8>(logits, labels, stats, coef, gout, dlogits, sh, 1, s);
    return launch_backward_at<T, 256, 4>(logits, labels, stats, coef, gout, dlogits, sh,
                                         ceil_div(n, 256 * 4), s);
  });
}

// The backward entry of every library.
inline int backward(const char* what, const void* logits, int dtype, const int64_t* labels,
                    const float* stats, const float* coef, const float* gout, void* dlogits,
                    int64_t B, int64_t S, int64_t V, int64_t bs, int64_t rs, int64_t ignore,
                    float temperature, hipStream_t stream) {
  Shape sh;
  int st = make_shape(B, S, V, bs, rs, ignore, temperature, dtype, &sh);
  if (st) return st;
  if (sh.rows == 0) return succeed();
  if (!logits || !labels || !stats || !coef || !dlogits)
    return fail(NL2K_ERR_NULL, "%s: a required pointer is NULL", what);
  if ((st = check_align(logits, dtype, "logits"))) return st;
  if ((st = check_align(dlogits, dtype, "dlogits"))) return st;
  if ((st = check_align(stats, kF32, "stats", 8))) return st;
  return launch_backward(logits, dtype, labels, reinterpret_cast<const f32x2*>(stats), coef, gout,
                         dlogits, sh, stream);
}

template <class T, int TPR, int K, class Op>
inline int launch_fused_at(const void* logits, const int64_t* labels, void* dlogits,
                           const Shape& sh, const Op& op, hipStream_t s) {
  unsigned grid;
  if (const int st = row_grid<TPR>(sh, 1, &grid)) return st;
  with_past<T>(sh, [&](auto past) {
    hipLaunchKernelGGL((fused_kernel<T, TPR, K, past(), Op>), dim3(grid), dim3(block_of<TPR>()), 0,
                       s, static_cast<const typename Elem<T>::type*>(logits), labels,
                       static_cast<typename Elem<T>::type*>(dlogits), sh, op);
  });
  return check_launch("fused_kernel");
}

// Rows that no registers hold take a workgroup of 1024, those below a window a wave.
template <class T, int TPR, class Op>
inline int launch_fused_long_at(const void* logits, const int64_t* labels, void* dlogits,
                                const Shape& sh, const Op& op, hipStream_t s) {
  unsigned grid;
  if (const int st = row_grid<TPR>(sh, 1, &grid)) return st;
  const bool past = bytes_of<T>(sh) > Caches::kGradient;
  auto* kernel = past ? &fused_long_kernel<T, TPR, 4, true, Op>
                      : &fused_long_kernel<T, TPR, 4, false, Op>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(block_of<TPR>()), 0, s,
                     static_cast<const typename Elem<T>::type*>(logits), labels,
                     static_cast<typename Elem<T>::type*>(dlogits), sh, op);
  return check_launch("fused_long_kernel");
}

// The fewest lanes whose registers hold a row, 16 windows each at most.
template <class Op>
inline int launch_fused(const void* logits, int dtype, const int64_t* labels, void* dlogits,
                        Shape sh, const Op& op, hipStream_t s) {
  return with_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int n = (sh.V + Elem<T>::E - 1) / Elem<T>::E;
    // what made the logits left its last rows in the caches, what reads the gradient begins with
    // the first: as quick alone, with such a reader 369 us against 396 at 512 MiB
    sh.last_first = true;
    if (sh.V < Elem<T>::E)
      return launch_fused_long_at<T, 64>(logits, labels, dlogits, sh, op, s);
    if (n > 16384) return launch_fused_long_at<T, 1024>(logits, labels, dlogits, sh, op, s);
    if (n <= 128) return launch_fused_at<T, 64, 2>(logits, labels, dlogits, sh, op, s);
    if (n <= 512) return launch_fused_at<T, 64, 8>(logits, labels, dlogits, sh, op, s);
    if (n <= 1024) return launch_fused_at<T, 256, 4>(logits, labels, dlogits, sh, op, s);
    if (n <= 2048) return launch_fused_at<T, 256, 8>(logits, labels, dlogits, sh, op, s);
    if (n <= 4096) return launch_fused_at<T, 256, 16>(logits, labels, dlogits, sh, op, s);
    if (n <= 8192) return launch_fused_at<T, 512, 16>(logits, labels, dlogits, sh, op, s);
    return launch_fused_at<T, 1024, 16>(logits, labels, dlogits, sh, op, s);
  });
}

}  // namespace rows
}  // namespace nl2k
