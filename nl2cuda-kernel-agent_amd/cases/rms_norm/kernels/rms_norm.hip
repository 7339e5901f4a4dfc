// Root-mean-square norm with the residual's addition, for MI355X (gfx950).
// C-ABI in include/rms_norm.h.
//
// A lane holds windows of eight numbers of a row, so that 16 lanes next to each
// other hold a block of 128; a wave, a workgroup of 256 or one of 1024 takes a
// row, which stays in registers from its sum of squares to its result.
//
// Bound by memory.  Measured with bfloat16 rows and a residual of the same type, where a large copy
// reaches 5.1 TB/s: 8192 x 4096 forward 47.0 us (5.7 TB/s of what it has to read and write),
// quantised 44.9 (5.2), backward 43.1 with dweight's second kernel (6.2); 4096 x 2048 11.7, 11.8 and
// 15.7; 16 x 4096 2.7, 3.1 and 5.3, which is a launch's latency and a few loads' (the backward has two
// launches).

#include "rms_norm.h"

#include "e4m3.h"

namespace {

using namespace nl2k::e4m3;

struct Forward {
  const void* x;
  const void* residual;
  const void* weight;
  void* y;        // numbers, or codes
  void* scales;
  void* h;
  float* rstd;
  int64_t x_stride, r_stride, pitch;
  int32_t rows, D;
  int w_dtype, scale_type;
  float eps;
};

// Eight weights.
__device__ __forceinline__ void weights8(const void* w, int dtype, int at, int count,
                                         float (&v)[8]) {
  if (dtype == kF32)
    values<float>(load8<float>(static_cast<const float*>(w) + at, count), v);
  else if (dtype == kBF16)
    values<bf16_t>(load8<bf16_t>(static_cast<const unsigned short*>(w) + at, count), v);
  else
    values<f16_t>(load8<f16_t>(static_cast<const unsigned short*>(w) + at, count), v);
}

// The sum over all TPR threads of a row; red has TPR / 64 floats.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = nl2k::wave_sum_dpp(v);
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v += red[i];
  }
  return v;
}

template <int TPR>
constexpr int block_of() {
  return TPR < 256 ? 256 : TPR;
}

template <int TPR>
__device__ __forceinline__ int row_in(int block) {
  return TPR == 64 ? block * 4 + (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : block;
}

template <int TPR>
__device__ __forceinline__ int lane_in() {
  return TPR == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
}

// h of a window: what is stored, widened again.
template <class T, class R, bool kRes>
__device__ __forceinline__ void sum8(const Raw<T>& x, const Raw<R>& r, float (&h)[8]) {
  values<T>(x, h);
  if constexpr (kRes) {
    float v[8];
    values<R>(r, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = widen<R>(narrow<R>(h[e] + v[e]));
  }
}

// y of a window at column k, from its h, of which `count` lie in the row.
template <class T, bool kCodes>
__device__ __forceinline__ void finish8(const Forward& f, int64_t row, int k, int count, float rstd,
                                        float (&v)[8], const float (&w)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd * w[e];
  if constexpr (kCodes) {
    const float top = nl2k::row16_max_dpp(magnitude(v));
    const Scale s =
        f.scale_type == kScaleF32 ? scale_of<kScaleF32>(top) : scale_of<kScaleE8M0>(top);
    u32x2 codes = pack8(v, s.inverse);
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // zeros behind the row, where 0 rstd = NaN too; 8192 x 4100 48.4 -> 49.1
      const int bits = 4 * max(min(count - 4 * i, 4), 0);  // half of them: no shift by 32
      codes[i] &= (1u << bits << bits) - 1;
    }
    if (count > 0 || k < (f.D + 15) / 16 * 16)
      *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(f.y) + row * f.pitch + k) = codes;
    if ((threadIdx.x & 15) == 0 && count > 0) {
      const int64_t at = (int64_t)(k / kBlock) * f.rows + row;
      if (f.scale_type == kScaleF32)
        keep<kScaleF32>(f.scales, at, s.kept);
      else
        keep<kScaleE8M0>(f.scales, at, s.kept);
    }
  } else {
    store8<T>(static_cast<typename Elem<T>::type*>(f.y) + row * f.D + k, count, v);
  }
}

// h = round(x + residual), y = h rstd weight with rstd = (mean(h^2) + eps)^(-1/2); all in 32 bits but
// for h, whose rounding to the residual's type is part of the function: a next layer reads that h.
//
// kWhole: rows are all of the windows, and nothing needs to ask where one ends, which saves a branch
// a load: 8192 x 4096 51.2 -> 47.8 us, 4096 x 2048 13.3 -> 11.7, its backward 16.6 -> 15.6.
template <class T, class R, bool kRes, bool kCodes, int TPR, int U, bool kWhole>
__global__ __launch_bounds__(block_of<TPR>()) void forward_kernel(Forward f) {
  __shared__ float red[TPR / 64];
  const int64_t row = row_in<TPR>(blockIdx.x);
  if (row >= f.rows) return;
  const int lane = lane_in<TPR>();
  const auto* x = static_cast<const typename Elem<T>::type*>(f.x) + row * f.x_stride;
  const auto* res = static_cast<const typename Elem<R>::type*>(f.residual) + row * f.r_stride;
  auto count = [&](int k) { return kWhole ? 8 : f.D - k; };
  Raw<T> xr[U];
  Raw<R> rr[kRes ? U : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    xr[u] = load8<T>(x + k, count(k));
    if constexpr (kRes) rr[u] = load8<R>(res + k, count(k));
  }
  float w[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    weights8(f.weight, f.w_dtype, k, count(k), w[u]);
  }
  float h[U][8], sum = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    sum8<T, R, kRes>(xr[u], rr[kRes ? u : 0], h[u]);
    if constexpr (kRes)
      store8<R>(static_cast<typename Elem<R>::type*>(f.h) + row * f.D + k, count(k), h[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[u][e], h[u][e], sum);
  }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(sum, red) / (float)f.D + f.eps);
  if (f.rstd && lane == 0) f.rstd[row] = rstd;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    finish8<T, kCodes>(f, row, k, count(k), rstd, h[u], w[u]);
  }
}

// Rows that registers do not hold, above 32768: read again for the result, mostly from the caches.
template <class T, class R, bool kRes, bool kCodes>
__global__ __launch_bounds__(1024) void forward_long_kernel(Forward f) {
  __shared__ float red[16];
  const int64_t row = blockIdx.x;
  const auto* x = static_cast<const typename Elem<T>::type*>(f.x) + row * f.x_stride;
  const auto* res = static_cast<const typename Elem<R>::type*>(f.residual) + row * f.r_stride;
  auto* hs = static_cast<typename Elem<R>::type*>(f.h) + row * f.D;
  auto load = [&](int k, float(&h)[8]) {
    const Raw<T> xr = load8<T>(x + k, f.D - k);
    Raw<R> rr{};
    if constexpr (kRes) rr = load8<R>(res + k, f.D - k);
    sum8<T, R, kRes>(xr, rr, h);
  };
  float sum = 0.f;
  for (int64_t c = threadIdx.x * 8; c < f.D; c += 8192) {
    const int k = (int)c;
    float h[8];
    load(k, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[e], h[e], sum);
  }
  const float rstd = 1.f / sqrtf(row_sum<1024>(sum, red) / (float)f.D + f.eps);
  if (f.rstd && threadIdx.x == 0) f.rstd[row] = rstd;
  // whole waves: the lanes of a block take their maximum together
  for (int64_t c = threadIdx.x * 8; c - threadIdx.x * 8 < f.D; c += 8192) {
    const int k = (int)min(c, (int64_t)INT32_MAX);
    float h[8], w[8];
    load(k, h);
    weights8(f.weight, f.w_dtype, k, f.D - k, w);
    if constexpr (kRes) store8<R>(hs + k, f.D - k, h);
    finish8<T, kCodes>(f, row, k, f.D - k, rstd, h, w);
  }
}

struct Backward {
  const void* dy;
  const void* h;
  const void* dh;
  const void* weight;
  const float* rstd;
  void* dx;
  void* dres;
  float* partial;  // [workgroups][D], null without a gradient of the weight
  int64_t dy_stride, h_stride, dh_stride;
  int32_t rows, D;
  int w_dtype;
};

// dx of a window, stored; u = h r in place of h, d = dy.
template <class T, class R>
__device__ __forceinline__ void gradient8(const Backward& b, int64_t row, int k, int count,
                                          float rstd, float mean, const float (&u)[8],
                                          const float (&d)[8], const float (&w)[8],
                                          const Raw<R>& dh) {
  float v[8], add[8];
  values<R>(dh, add);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = fmaf(rstd, d[e] * w[e] - u[e] * mean, add[e]);
  if (b.dx) store8<T>(static_cast<typename Elem<T>::type*>(b.dx) + row * b.D + k, count, v);
  if (b.dres) store8<R>(static_cast<typename Elem<R>::type*>(b.dres) + row * b.D + k, count, v);
}

// With d = dy, u = h rstd and c = mean(d weight u) over the row:
//   dx = dresidual = rstd (d weight - u c) + dh,  dweight = sum over rows of d u.
// A workgroup takes every gridDim.x-th row (or four), and adds up their share of dweight in registers;
// columns_kernel adds the workgroups' shares, so that no atomics are needed and the order is fixed.
// dh and rows' ends are asked for before they are loaded, not masked out of a load: without a
// residual 16384 x 2048 56 -> 47 us, 65536 x 256 49 -> 34.  Loading the next row ahead gave nothing
// where the other workgroups of a CU cover the wait; one of 1024 threads has its CU to itself, and its
// rows' loads and sums follow one another: 999 x 5121 float32 14.3 us, its bytes 12.
template <class T, class R, int TPR, int U, bool kWhole>
__global__ __launch_bounds__(block_of<TPR>()) void backward_kernel(Backward b) {
  constexpr int kRows = block_of<TPR>() / TPR;
  __shared__ float red[TPR / 64];
  __shared__ float shared_dw[kRows > 1 ? TPR * U * 8 : 1];
  const int lane = lane_in<TPR>();
  auto count = [&](int k) { return kWhole ? 8 : b.D - k; };
  float w[U][8], dw[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    weights8(b.weight, b.w_dtype, k, count(k), w[u]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[u][e] = 0.f;
  }
  for (int64_t row = row_in<TPR>(blockIdx.x); row < b.rows; row += (int64_t)gridDim.x * kRows) {
    const auto* dy = static_cast<const typename Elem<T>::type*>(b.dy) + row * b.dy_stride;
    const auto* h = static_cast<const typename Elem<R>::type*>(b.h) + row * b.h_stride;
    const auto* dh = static_cast<const typename Elem<R>::type*>(b.dh) + row * b.dh_stride;
    Raw<T> dr[U];
    Raw<R> hr[U], ar[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (u * TPR + lane) * 8;
      dr[u] = load8<T>(dy + k, count(k));
      hr[u] = load8<R>(h + k, count(k));
      ar[u] = Raw<R>{};
      if (b.dh) ar[u] = load8<R>(dh + k, count(k));
    }
    const float rstd = b.rstd[row];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float d[8], v[8];
      values<T>(dr[u], d);
      values<R>(hr[u], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] *= rstd;
        sum = fmaf(d[e] * w[u][e], v[e], sum);
        dw[u][e] = fmaf(d[e], v[e], dw[u][e]);
      }
    }
    const float mean = row_sum<TPR>(sum, red) / (float)b.D;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float d[8], v[8];
      values<T>(dr[u], d);
      values<R>(hr[u], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= rstd;
      const int k = (u * TPR + lane) * 8;
      gradient8<T, R>(b, row, k, count(k), rstd, mean, v, d, w[u], ar[u]);
    }
  }
  if (!b.partial) return;
  if constexpr (kRows > 1) {  // the waves' sums, added in their order
    for (int i = 0; i < kRows; ++i) {
      if (i) __syncthreads();
      if ((int)(threadIdx.x >> 6) != i) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float* at = shared_dw + (u * 8 + e) * 64 + lane;
          dw[u][e] += i ? *at : 0.f;
          *at = dw[u][e];
        }
    }
    if ((int)(threadIdx.x >> 6) != kRows - 1) return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = (u * TPR + lane) * 8;
    store8<float>(b.partial + (int64_t)blockIdx.x * b.D + k, count(k), dw[u]);
  }
}

// Rows above 16384, whose share of dweight registers do not hold: in the workgroup's own row of the
// workspace, added to at each of its rows; 1024 x 32768 103 us (2.6 TB/s of what the others move).
template <class T, class R>
__global__ __launch_bounds__(1024) void backward_long_kernel(Backward b) {
  __shared__ float red[16];
  float* mine = b.partial ? b.partial + (int64_t)blockIdx.x * b.D : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < b.rows; row += gridDim.x) {
    const auto* dy = static_cast<const typename Elem<T>::type*>(b.dy) + row * b.dy_stride;
    const auto* h = static_cast<const typename Elem<R>::type*>(b.h) + row * b.h_stride;
    const auto* dh = static_cast<const typename Elem<R>::type*>(b.dh) + row * b.dh_stride;
    const float rstd = b.rstd[row];
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < b.D; c += 8192) {
      const int k = (int)c;
      float d[8], v[8], w[8];
      values<T>(load8<T>(dy + k, b.D - k), d);
      values<R>(load8<R>(h + k, b.D - k), v);
      weights8(b.weight, b.w_dtype, k, b.D - k, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(d[e] * w[e], v[e] * rstd, sum);
    }
    const float mean = row_sum<1024>(sum, red) / (float)b.D;
    for (int64_t c = threadIdx.x * 8; c < b.D; c += 8192) {
      const int k = (int)c;
      float d[8], v[8], w[8];
      values<T>(load8<T>(dy + k, b.D - k), d);
      values<R>(load8<R>(h + k, b.D - k), v);
      weights8(b.weight, b.w_dtype, k, b.D - k, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= rstd;
      if (mine) {  // this thread's columns alone
        float p[8];
        values<float>(load8<float>(mine + k, first ? 0 : b.D - k), p);
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = fmaf(d[e], v[e], p[e]);
        store8<float>(mine + k, b.D - k, p);
      }
      Raw<R> add{};
      if (b.dh) add = load8<R>(dh + k, b.D - k);
      gradient8<T, R>(b, row, k, b.D - k, rstd, mean, v, d, w, add);
    }
    first = false;
  }
}

// dweight: the workgroups' sums, 16 columns a workgroup, from column `first` on, 16 threads a column.
__global__ __launch_bounds__(256) void columns_kernel(const float* __restrict__ partial, int count,
                                                      int D, int first, void* dw, int w_dtype) {
  __shared__ float part[16][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t col = first + (int64_t)blockIdx.x * 16 + c;
  float sum = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int i = g; i < count; i += 16) sum += partial[(int64_t)i * D + col];
  }
  part[g][c] = sum;
  __syncthreads();
  if (g == 0 && col < D) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += part[i][c];
    if (w_dtype == kF32)
      static_cast<float*>(dw)[col] = s;
    else
      static_cast<unsigned short*>(dw)[col] =
          w_dtype == kBF16 ? narrow<bf16_t>(s) : narrow<f16_t>(s);
  }
}

// Threads a row and windows a thread for a row of D numbers.  The fewest threads that hold a row lose
// least to its sum, more of them have more loads in the air.  bfloat16 with a residual, forward and
// backward in us, against the neighbour that also holds the row:
//   1024: {64, 2} 47.2, 42.5 (32768 rows);   {256, 1} 52.4, 81.7
//   2048: {256, 1} 11.7, 15.7 (4096 rows);   {64, 4} 12.8, 16.8
//   4096: {256, 2} 47.0, 43.1 (8192 rows);   {1024, 1} 52.3, 56.2
//   8192: {1024, 1} 21.8, 24.5 (2048 rows);  {256, 4} 23.0, 28.0
//   16384: {1024, 2} 50.0, 51.2 (2048 rows); {256, 8} 52.7, 68.0
struct Plan {
  int tpr, u;
};

Plan plan(int64_t D) {
  const int64_t n = nl2k::ceil_div(D, 8);
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return {256, 1};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {1024, 1};
  if (n <= 2048) return {1024, 2};
  if (n <= 4096) return {1024, 4};
  return {0, 0};
}

// Workgroups of a backward: each has a row of the workspace that the second kernel reads, and must be
// enough of them to have the memory busy.  Rows of up to 256 numbers leave most of a wave's lanes idle:
// 65536 x 256 33.6 us with 512 workgroups, 27.8 with 1024, where 8192 x 4096 has 43.4 and 48.9.
// Workgroups of 1024 threads are one a CU: 999 x 5121 float32 18.8 with 256, 21.9 with 512, 2048 x
// 16384 51.8 and 60.1.
int64_t backward_blocks(int64_t rows, int64_t D) {
  const Plan p = plan(D);
  const int64_t most = p.tpr == 1024 || p.tpr == 0 ? 256 : D <= 256 ? 1024 : 512;
  return std::min(p.tpr == 64 ? nl2k::ceil_div(rows, 4) : rows, most);
}

template <class F>
int with_types(int dtype, int r_dtype, F&& f) {
  if (dtype == kF32) return f(float{}, float{});
  if (dtype == kBF16) return r_dtype == kF32 ? f(bf16_t{}, float{}) : f(bf16_t{}, bf16_t{});
  return r_dtype == kF32 ? f(f16_t{}, float{}) : f(f16_t{}, f16_t{});
}

template <class T, class R, bool kRes, bool kCodes, bool kWhole>
void pick_forward(const Plan& p, const Forward& f, dim3 grid, hipStream_t s) {
  auto is = [&](int t, int u) { return p.tpr == t && p.u == u; };
  if (is(64, 1))
    forward_kernel<T, R, kRes, kCodes, 64, 1, kWhole><<<grid, 256, 0, s>>>(f);
  else if (is(64, 2))
    forward_kernel<T, R, kRes, kCodes, 64, 2, kWhole><<<grid, 256, 0, s>>>(f);
  else if (is(256, 1))
    forward_kernel<T, R, kRes, kCodes, 256, 1, kWhole><<<grid, 256, 0, s>>>(f);
  else if (is(256, 2))
    forward_kernel<T, R, kRes, kCodes, 256, 2, kWhole><<<grid, 256, 0, s>>>(f);
  else if (is(1024, 1))
    forward_kernel<T, R, kRes, kCodes, 1024, 1, kWhole><<<grid, 1024, 0, s>>>(f);
  else if (is(1024, 2))
    forward_kernel<T, R, kRes, kCodes, 1024, 2, kWhole><<<grid, 1024, 0, s>>>(f);
  else
    forward_kernel<T, R, kRes, kCodes, 1024, 4, kWhole><<<grid, 1024, 0, s>>>(f);
}

// More rows than a launch has workgroups go in several.
template <class T, class R, bool kRes, bool kCodes>
int launch_forward(Forward f, hipStream_t s) {
  const Plan p = plan(f.D);
  const int64_t most = p.tpr == 64 ? f.rows : nl2k::max_blocks(p.tpr == 256 ? 256 : 1024);
  for (int64_t left = f.rows;;) {
    const int64_t n = std::min(left, most);
    const dim3 grid((uint32_t)(p.tpr == 64 ? nl2k::ceil_div(n, 4) : n));
    if (p.tpr == 0)
      forward_long_kernel<T, R, kRes, kCodes><<<grid, 1024, 0, s>>>(f);
    else if (f.D == p.tpr * p.u * 8)
      pick_forward<T, R, kRes, kCodes, true>(p, f, grid, s);
    else
      pick_forward<T, R, kRes, kCodes, false>(p, f, grid, s);
    if (int st = nl2k::check_launch("rms_norm")) return st;
    if ((left -= n) == 0) return NL2K_SUCCESS;
    // scales lie blocks first: f.rows stays the number of all rows
    auto on = [](const void* p, int64_t bytes) { return static_cast<const char*>(p) + bytes; };
    f.x = on(f.x, n * f.x_stride * Elem<T>::bytes);
    if (kRes) f.residual = on(f.residual, n * f.r_stride * Elem<R>::bytes);
    if (kRes) f.h = const_cast<char*>(on(f.h, n * f.D * Elem<R>::bytes));
    f.y = const_cast<char*>(on(f.y, kCodes ? n * f.pitch : n * f.D * Elem<T>::bytes));
    if (kCodes) f.scales = const_cast<char*>(on(f.scales, n * scale_bytes(f.scale_type)));
    if (f.rstd) f.rstd += n;
  }
}

template <class T, class R, bool kWhole>
void pick_backward(const Plan& p, const Backward& b, dim3 grid, hipStream_t s) {
  auto is = [&](int t, int u) { return p.tpr == t && p.u == u; };
  if (is(64, 1))
    backward_kernel<T, R, 64, 1, kWhole><<<grid, 256, 0, s>>>(b);
  else if (is(64, 2))
    backward_kernel<T, R, 64, 2, kWhole><<<grid, 256, 0, s>>>(b);
  else if (is(256, 1))
    backward_kernel<T, R, 256, 1, kWhole><<<grid, 256, 0, s>>>(b);
  else if (is(256, 2))
    backward_kernel<T, R, 256, 2, kWhole><<<grid, 256, 0, s>>>(b);
  else if (is(1024, 1))
    backward_kernel<T, R, 1024, 1, kWhole><<<grid, 1024, 0, s>>>(b);
  else
    backward_kernel<T, R, 1024, 2, kWhole><<<grid, 1024, 0, s>>>(b);
}

template <class T, class R>
int launch_backward(const Backward& b, hipStream_t s) {
  const Plan p = plan(b.D);
  const dim3 grid((uint32_t)backward_blocks(b.rows, b.D));
  if (p.tpr == 0 || p.tpr * p.u > 2048)
    backward_long_kernel<T, R><<<grid, 1024, 0, s>>>(b);
  else if (b.D == p.tpr * p.u * 8)
    pick_backward<T, R, true>(p, b, grid, s);
  else
    pick_backward<T, R, false>(p, b, grid, s);
  return nl2k::check_launch("rms_norm_backward");
}

// Sizes and types that all entries share.
int check_sizes(const char* who, int64_t rows, int64_t D, int dtype, int r_dtype, int w_dtype) {
  if (rows < 0 || D < 1)
    return nl2k::fail(NL2K_ERR_SHAPE, "%s: need rows >= 0 and D >= 1 (got %lld, %lld)", who,
                      (long long)rows, (long long)D);
  // four rows a workgroup of 256 threads in one launch
  if (D > INT32_MAX - 16384 || rows > 4 * nl2k::max_blocks(256))
    return nl2k::fail(NL2K_ERR_OVERFLOW, "%s: sizes too large (rows=%lld D=%lld)", who,
                      (long long)rows, (long long)D);
  if (dtype < kF32 || dtype > kF16 || w_dtype < kF32 || w_dtype > kF16 ||
      (r_dtype != dtype && r_dtype != kF32))
    return nl2k::fail(NL2K_ERR_VALUE,
                      "%s: types must be 0, 1 or 2, the residual's that of x or 0 (got %d, %d, %d)",
                      who, dtype, r_dtype, w_dtype);
  return NL2K_SUCCESS;
}

int check_rows(const char* who, const char* name, const void* p, int dtype, int64_t stride,
               int64_t rows) {
  if (reinterpret_cast<uintptr_t>(p) % bytes_of(dtype))
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: %s must be aligned to its type", who, name);
  if (stride < 0 || (rows > 1 && stride > INT64_MAX / 8 / rows))
    return nl2k::fail(NL2K_ERR_SHAPE, "%s: the stride of %s is negative or too large (%lld)", who,
                      name, (long long)stride);
  return NL2K_SUCCESS;
}

int forward(const char* who, Forward f, int dtype, int r_dtype, bool codes, int64_t rows,
            int64_t D, hipStream_t stream) {
  int st = check_sizes(who, rows, D, dtype, f.residual ? r_dtype : dtype, f.w_dtype);
  if (st) return st;
  if (!(f.eps > 0.f && f.eps <= 3.4e38f))
    return nl2k::fail(NL2K_ERR_VALUE, "%s: eps must be positive and finite", who);
  if (codes && f.scale_type != kScaleF32 && f.scale_type != kScaleE8M0)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: scale_type must be 0 or 1 (got %d)", who, f.scale_type);
  if (rows == 0) return nl2k::succeed();
  if (!f.x || !f.weight || !f.y || (codes && !f.scales) || !f.residual != !f.h)
    return nl2k::fail(NL2K_ERR_NULL,
                      "%s: x, weight and the output are required, residual and h together", who);
  if ((st = check_rows(who, "x", f.x, dtype, f.x_stride, rows))) return st;
  if ((st = check_rows(who, "residual", f.residual, r_dtype, f.r_stride, rows))) return st;
  if ((st = check_rows(who, "h", f.h, r_dtype, 0, rows))) return st;
  if ((st = check_rows(who, "weight", f.weight, f.w_dtype, 0, rows))) return st;
  if ((st = check_rows(who, "rstd", f.rstd, kF32, 0, rows))) return st;
  if (codes) {
    if (f.pitch < D || f.pitch % 16 || f.pitch > INT64_MAX / 8 / rows)
      return nl2k::fail(NL2K_ERR_SHAPE, "%s: the pitch of codes must be >= D, a multiple of 16",
                        who);
    if (!nl2k::aligned16(f.y) ||
        reinterpret_cast<uintptr_t>(f.scales) % scale_bytes(f.scale_type))
      return nl2k::fail(NL2K_ERR_ALIGN, "%s: codes must be aligned to 16 bytes, scales to their type",
                        who);
  } else if ((st = check_rows(who, "y", f.y, dtype, 0, rows))) {
    return st;
  }
  f.rows = (int32_t)rows;
  f.D = (int32_t)D;
  return with_types(dtype, f.residual ? r_dtype : dtype, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    if (f.residual)
      return codes ? launch_forward<T, R, true, true>(f, stream)
                   : launch_forward<T, R, true, false>(f, stream);
    if constexpr (__is_same(T, R))
      return codes ? launch_forward<T, T, false, true>(f, stream)
                   : launch_forward<T, T, false, false>(f, stream);
    return nl2k::succeed();  // not reached: without a residual the types agree
  });
}

}  // namespace

extern "C" int rms_norm_forward(const void* x, int dtype, int64_t x_stride, const void* residual,
                                int residual_dtype, int64_t residual_stride, const void* weight,
                                int weight_dtype, void* y, void* h, float* rstd, int64_t rows,
                                int64_t D, float eps, hipStream_t stream) {
  const Forward f{x,  residual, weight,          y, nullptr, h, rstd, x_stride, residual_stride,
                  0,  0,        0, weight_dtype, 0, eps};
  return forward("rms_norm_forward", f, dtype, residual_dtype, false, rows, D, stream);
}

extern "C" int rms_norm_quant(const void* x, int dtype, int64_t x_stride, const void* residual,
                              int residual_dtype, int64_t residual_stride, const void* weight,
                              int weight_dtype, void* codes, int64_t pitch, void* scales,
                              int scale_type, void* h, int64_t rows, int64_t D, float eps,
                              hipStream_t stream) {
  const Forward f{x,     residual, weight, codes, scales, h, nullptr, x_stride, residual_stride,
                  pitch, 0,        0,      weight_dtype, scale_type, eps};
  return forward("rms_norm_quant", f, dtype, residual_dtype, true, rows, D, stream);
}

extern "C" size_t rms_norm_backward_workspace_bytes(int64_t rows, int64_t D) {
  if (check_sizes("rms_norm_backward_workspace_bytes", rows, D, kF32, kF32, kF32)) return 0;
  return (size_t)backward_blocks(rows, D) * D * 4;
}

extern "C" int rms_norm_backward(const void* dy, int dtype, int64_t dy_stride, const void* h,
                                 int h_dtype, int64_t h_stride, const void* dh, int64_t dh_stride,
                                 const void* weight, int weight_dtype, const float* rstd, void* dx,
                                 void* dresidual, void* dweight, int64_t rows, int64_t D,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const char* who = "rms_norm_backward";
  int st = check_sizes(who, rows, D, dtype, h_dtype, weight_dtype);
  if (st) return st;
  if (rows && (!dy || !h || !weight || !rstd))
    return nl2k::fail(NL2K_ERR_NULL, "%s: dy, h, weight and rstd are required", who);
  if ((st = check_rows(who, "dy", dy, dtype, dy_stride, rows))) return st;
  if ((st = check_rows(who, "h", h, h_dtype, h_stride, rows))) return st;
  if ((st = check_rows(who, "dh", dh, h_dtype, dh_stride, rows))) return st;
  if ((st = check_rows(who, "weight", weight, weight_dtype, 0, rows))) return st;
  if ((st = check_rows(who, "rstd", rstd, kF32, 0, rows))) return st;
  if ((st = check_rows(who, "dx", dx, dtype, 0, rows))) return st;
  if ((st = check_rows(who, "dresidual", dresidual, h_dtype, 0, rows))) return st;
  if ((st = check_rows(who, "dweight", dweight, weight_dtype, 0, rows))) return st;
  const size_t need = dweight ? (size_t)backward_blocks(rows, D) * D * 4 : 0;
  if (need && (!workspace || workspace_bytes < need))
    return nl2k::fail(NL2K_ERR_WORKSPACE, "%s: needs a workspace of %zu bytes (got %zu)", who, need,
                      workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 4)
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: the workspace must be aligned to 4 bytes", who);
  const Backward b{dy, h, dh, weight, rstd, dx, dresidual,
                   dweight ? static_cast<float*>(workspace) : nullptr, dy_stride, h_stride,
                   dh_stride, (int32_t)rows, (int32_t)D, weight_dtype};
  if (rows) {
    st = with_types(dtype, h_dtype, [&](auto t, auto r) {
      return launch_backward<decltype(t), decltype(r)>(b, stream);
    });
    if (st) return st;
  }
  if (dweight) {
    const int count = rows ? (int)backward_blocks(rows, D) : 0;
    // 2^28 columns and more have more workgroups than a launch
    const int64_t most = 16 * nl2k::max_blocks(256);
    for (int64_t first = 0; first < D; first += most) {
      const int64_t n = nl2k::ceil_div(std::min(D - first, most), 16);
      columns_kernel<<<dim3((uint32_t)n), 256, 0, stream>>>(b.partial, count, (int)D, (int)first,
                                                            dweight, weight_dtype);
      if ((st = nl2k::check_launch(who))) return st;
    }
    return st;
  }
  return nl2k::succeed();
}

extern "C" const char* rms_norm_last_error(void) { return nl2k::error_slot().text; }
