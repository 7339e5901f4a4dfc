// Orthogonalised updates by Newton-Schulz products, for MI355X (gfx950).
// C-ABI in include/newton_schulz.h.
//
// With k = min(m, n) and l = max(m, n), X is held as [k, l] and its transpose
// [l, k], so that all three products of a step are of one form, rows by rows:
//
//   A  = X X'            [k, k], symmetric: tiles on and below the diagonal
//   B  = b A + c A A'    [k, k], symmetric (A = A')
//   X  = a X + B (X')'   [k, l]; written as X and as X'
//
// Operands are float16 times a power of two (kept by the host from bounds on
// the singular values), accumulators float32.  In full precision an operand
// is a sum of two float16, and a product the three larger ones of its four:
// 22 bits.  The two halves of 32 elements along a row lie next to each other,
// so a tile is loaded alike in both precisions.

#include "newton_schulz.h"

#include <cmath>

#include "common.h"
#include "lds_direct.h"

namespace {

using nl2k::f32x4;
using nl2k::u32x4;
using namespace nl2k::lds;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half_t;

constexpr int kBatch = 32;        // matrices of one launch: their pointers are kernel arguments
constexpr int kPartials = 1024;   // most workgroups that sum a matrix's squares
constexpr int kStep = 64;         // float16 of a row that a stage takes: 128 bytes
constexpr size_t kMaxBatchBytes = (size_t)4 << 30;

// ------------------------------------------------------------------ elements
// Eight elements of a user's matrix at any alignment of its own type; of the
// last ones of a row `count` < 8.
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float widen(unsigned short h, int dtype) {
  return dtype == 1 ? __builtin_bit_cast(float, (uint32_t)h << 16)
                    : (float)__builtin_bit_cast(half_t, h);
}

__device__ __forceinline__ unsigned short narrow(float v, int dtype) {
  return dtype == 1 ? __builtin_bit_cast(unsigned short, (__bf16)v)
                    : __builtin_bit_cast(unsigned short, (half_t)v);
}

__device__ __forceinline__ void load8(const void* p, int64_t at, int dtype, int count,
                                      float (&v)[8]) {
  if (dtype == 0) {
    const float* q = static_cast<const float*>(p) + at;
    if (count >= 8) {
      const f32x4 a = *reinterpret_cast<const f32x4_u*>(q);
      const f32x4 b = *reinterpret_cast<const f32x4_u*>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < count ? q[e] : 0.f;
    }
  } else {
    const unsigned short* q = static_cast<const unsigned short*>(p) + at;
    u16x8 h;
    if (count >= 8) {
      h = __builtin_bit_cast(u16x8, (u32x4)*reinterpret_cast<const u32x4_u*>(q));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = e < count ? q[e] : (unsigned short)0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widen(h[e], dtype);
  }
}

__device__ __forceinline__ void store8(void* p, int64_t at, int dtype, int count,
                                       const float (&v)[8]) {
  if (dtype == 0) {
    float* q = static_cast<float*>(p) + at;
    if (count >= 8) {
      *reinterpret_cast<f32x4_u*>(q) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_u*>(q + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) q[e] = v[e];
    }
  } else {
    unsigned short* q = static_cast<unsigned short*>(p) + at;
    u16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = narrow(v[e], dtype);
    if (count >= 8) {
      *reinterpret_cast<u32x4_u*>(q) = __builtin_bit_cast(u32x4, h);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) q[e] = h[e];
    }
  }
}

__device__ __forceinline__ float load1(const void* p, int64_t at, int dtype) {
  return dtype == 0 ? static_cast<const float*>(p)[at]
                    : widen(static_cast<const unsigned short*>(p)[at], dtype);
}

__device__ __forceinline__ void store1(void* p, int64_t at, int dtype, float v) {
  if (dtype == 0)
    static_cast<float*>(p)[at] = v;
  else
    static_cast<unsigned short*>(p)[at] = narrow(v, dtype);
}

// Eight elements t .. t + 7 of an operand row, t a multiple of 8: in full
// precision the second halves lie 32 on.
template <int PL>
struct Halves {
  f16x8 h[PL];
};

template <int PL>
__device__ __forceinline__ int64_t at(int t) {
  return PL == 1 ? t : (int64_t)(t >> 5) * 64 + (t & 31);
}

template <int PL>
__device__ __forceinline__ Halves<PL> get8(const half_t* row, int t) {
  Halves<PL> r;
#pragma unroll
  for (int p = 0; p < PL; ++p)
    r.h[p] = *reinterpret_cast<const f16x8*>(row + at<PL>(t) + 32 * p);
  return r;
}

template <int PL>
__device__ __forceinline__ float value(const Halves<PL>& r, int e) {
  return PL == 2 ? (float)r.h[0][e] + (float)r.h[PL - 1][e] : (float)r.h[0][e];
}

template <int PL>
__device__ __forceinline__ void put8(half_t* row, int t, const float (&v)[8]) {
  f16x8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = (half_t)v[e];
    lo[e] = (half_t)(v[e] - (float)hi[e]);
  }
  half_t* p = row + at<PL>(t);
  *reinterpret_cast<f16x8*>(p) = hi;
  if (PL == 2) *reinterpret_cast<f16x8*>(p + 32) = lo;
}

// ------------------------------------------------------------------ prologue
struct Source {
  const void* g[kBatch];
  void* mom[kBatch];  // null without a momentum
  int g_dtype, m_dtype;
  int64_t g_stride, m_stride;
  float mu;
  int nesterov;
  int m, n;
};

// U from G and the momentum after its update.
__device__ __forceinline__ void update_of(const Source& s, float (&g)[8], const float (&mom)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = s.nesterov ? fmaf(s.mu, mom[e], g[e]) : mom[e];
}

// Momentum and the sum of U's squares, a partial sum in 64 bits a workgroup:
// the squares of 32-bit numbers leave 32 bits on either side.
__global__ __launch_bounds__(256) void square_kernel(Source s, double* __restrict__ partial) {
  __shared__ double red[4];
  const int b = blockIdx.y;
  const void* g = s.g[b];
  void* mom = s.mom[b];
  const int groups = (s.n + 7) / 8;  // of eight elements a row
  const int64_t total = (int64_t)groups * s.m;
  double sum = 0.0;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total;
       x += (int64_t)gridDim.x * 256) {
    const int i = total < (int64_t)1 << 31 ? (uint32_t)x / (uint32_t)groups : (int)(x / groups);
    const int j = (int)(x - (int64_t)i * groups) * 8;
    float u[8];
    load8(g, i * s.g_stride + j, s.g_dtype, s.n - j, u);
    if (mom) {
      const int64_t at_m = i * s.m_stride + j;
      float v[8];
      load8(mom, at_m, s.m_dtype, s.n - j, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = fmaf(s.mu, v[e], u[e]);
        // as it is kept, so that U is what a reader of the momentum would form
        if (s.m_dtype != 0) v[e] = widen(narrow(v[e], s.m_dtype), s.m_dtype);
      }
      store8(mom, at_m, s.m_dtype, s.n - j, v);
      update_of(s, u, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (double)u[e] * u[e];
  }
  sum = nl2k::wave_sum(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    partial[(int64_t)b * kPartials + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X_0 and its transpose, times sx, from U: 64 x 64 tiles through LDS.  Rows of
// both are padded with zeros to a multiple of a tile step.
template <int PL>
__global__ __launch_bounds__(256) void scale_kernel(Source s, const double* __restrict__ partial,
                                                    int blocks, float eps, float sx,
                                                    half_t* __restrict__ rows, int rows_pitch,
                                                    int rows_len, int64_t rows_batch,
                                                    half_t* __restrict__ cols, int cols_pitch,
                                                    int cols_len, int64_t cols_batch) {
  __shared__ float tile[64][68];
  __shared__ double red[4];
  const int b = blockIdx.z;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  float u[2][8];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = i0 + (threadIdx.x >> 3) + 32 * q, j = j0 + (threadIdx.x & 7) * 8;
    const int count = i < s.m ? s.n - j : 0;
    if (count > 0) {
      load8(s.g[b], i * s.g_stride + j, s.g_dtype, count, u[q]);
      if (s.mom[b]) {
        float v[8];
        load8(s.mom[b], i * s.m_stride + j, s.m_dtype, count, v);
        update_of(s, u[q], v);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) u[q][e] = e < count ? u[q][e] : 0.f;
  }
  double part = 0.0;
  for (int x = threadIdx.x; x < blocks; x += 256) part += partial[(int64_t)b * kPartials + x];
  part = nl2k::wave_sum(part);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = part;
  __syncthreads();
  const double f = sqrt((red[0] + red[1]) + (red[2] + red[3])) + (double)eps;
  // 0 / 0 is an update of zeros; sx / f may pass 32 bits where the elements are small
  const double scale = f > 0.0 ? sx / f : (f == 0.0 ? 0.0 : NAN);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = (threadIdx.x >> 3) + 32 * q, c = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[q][e] = (float)(u[q][e] * scale);
      tile[r][c + e] = u[q][e];
    }
    // rows: [m, n] padded along n to rows_len, cols: [n, m] along m to cols_len
    if (i0 + r < s.m && j0 + c < rows_len)
      put8<PL>(rows + b * rows_batch + (int64_t)(i0 + r) * rows_pitch, j0 + c, u[q]);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int c = (threadIdx.x >> 3) + 32 * q, r = (threadIdx.x & 7) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r + e][c];
    if (j0 + c < s.n && i0 + r < cols_len)
      put8<PL>(cols + b * cols_batch + (int64_t)(j0 + c) * cols_pitch, i0 + r, v);
  }
}

// ------------------------------------------------------------------ products
// acc(i, j) = sum_t P[i, t] Q[j, t] for one tile.
struct Operands {
  const half_t* p;
  const half_t* q;
  int p_rows, q_rows;
  int p_pitch, q_pitch;      // float16 a row
  int64_t p_batch, q_batch;  // float16 a matrix
  int row_bytes;             // of a row, padded
  int steps;                 // stages that those are
  int tiles_p, tiles_q;      // tiles of a matrix
  int tiles;                 // all of them
};

// What becomes of the sums.  row8 is given eight of a row, turns them into the
// result and stores it; col8 is given eight of the result down a column, where
// a transpose is stored too.  `Pre` is what row8 reads from memory, fetched
// ahead of the sums.

// A symmetric result [n, n], both triangles from the tiles on and below the
// diagonal: v = alpha acc + beta D.
template <int PL>
struct SymmetricStore {
  static constexpr bool kSymmetric = true;
  static constexpr bool kSplit = false;
  half_t* c;
  const half_t* d;
  int n, pitch, cols;  // cols: n padded to a tile step
  int64_t batch;
  float alpha, beta;
  using Pre = Halves<PL>;
  __device__ __forceinline__ Pre fetch(int b, int i, int j) const {
    Pre r{};
    if (d && i < n && j < cols) r = get8<PL>(d + b * batch + (int64_t)i * pitch, j);
    return r;
  }
  __device__ __forceinline__ void row8(int b, int i, int j, float (&v)[8], const Pre& pre) const {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = i < n && j + e < n ? fmaf(beta, value<PL>(pre, e), alpha * v[e]) : 0.f;
    if (i < n && j < cols) put8<PL>(c + b * batch + (int64_t)i * pitch, j, v);
  }
  __device__ __forceinline__ bool columns(bool diagonal) const { return !diagonal; }
  __device__ __forceinline__ void col8(int b, int i, int j, const float (&v)[8]) const {
    if (j < n && i < cols) put8<PL>(c + b * batch + (int64_t)j * pitch, i, v);
  }
};

// One part of the sums of a symmetric product, along its rows: 64 x 64 tiles of
// float32, one after the other, for sum_kernel to add.
constexpr int kSplitTile = 64 * 64;
constexpr int kSplitTiles = 512;  // most of them, all parts together
struct SplitStore {
  static constexpr bool kSymmetric = true;
  static constexpr bool kSplit = true;
  float* parts;
  int nb, per;  // matrices; stages of a part
  int tiles;    // of a matrix
  struct Pre {};
  __device__ __forceinline__ Pre fetch(int, int, int) const { return Pre{}; }
  __device__ __forceinline__ void row8(int b, int i, int j, float (&v)[8], const Pre&) const {
    const int ti = i >> 6, tj = j >> 6;
    float* q = parts + ((int64_t)b * tiles + ti * (ti + 1) / 2 + tj) * kSplitTile +
               (i & 63) * 64 + (j & 63);
    *reinterpret_cast<f32x4*>(q) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(q + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
  __device__ __forceinline__ bool columns(bool) const { return false; }
  __device__ __forceinline__ void col8(int, int, int, const float (&)[8]) const {}
};

// The parts of a symmetric product, added in their order and stored.
template <int PL>
__global__ __launch_bounds__(256) void sum_kernel(const float* __restrict__ parts, int count,
                                                  SymmetricStore<PL> store) {
  __shared__ float tile[64][68];
  const int tiles = gridDim.x, nb = gridDim.y, b = blockIdx.y;
  int ti = 0;
  while ((ti + 1) * (ti + 2) / 2 <= (int)blockIdx.x) ++ti;
  const int tj = blockIdx.x - ti * (ti + 1) / 2;
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
  f32x4 sum[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) sum[q] = nl2k::zero4();
#pragma unroll 4
  for (int s = 0; s < count; ++s) {
    const float* p =
        parts + (((int64_t)s * nb + b) * tiles + blockIdx.x) * kSplitTile + r * 64 + c;
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] += nl2k::load4(p + 4 * q);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 lo = sum[2 * h], hi = sum[2 * h + 1];
    float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    const int i = ti * 64 + r, j = tj * 64 + c + 8 * h;
    store.row8(b, i, j, v, store.fetch(b, i, j));
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[r][c + 8 * h + e] = v[e];
  }
  __syncthreads();
  if (!store.columns(ti == tj)) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int col = threadIdx.x >> 2, row = ((threadIdx.x & 3) * 2 + h) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[row + e][col];
    store.col8(b, ti * 64 + row, tj * 64 + col, v);
  }
}

// X = alpha acc + beta X, as [k, l] in place and as [l, k].
template <int PL>
struct StepStore {
  static constexpr bool kSymmetric = false;
  static constexpr bool kSplit = false;
  half_t* x;
  half_t* xt;
  int k, l, x_pitch, t_pitch, x_cols, t_cols;
  int64_t x_batch, t_batch;
  float alpha, beta;
  using Pre = Halves<PL>;
  __device__ __forceinline__ Pre fetch(int b, int i, int j) const {
    Pre r{};
    if (i < k && j < x_cols) r = get8<PL>(x + b * x_batch + (int64_t)i * x_pitch, j);
    return r;
  }
  __device__ __forceinline__ void row8(int b, int i, int j, float (&v)[8], const Pre& pre) const {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = i < k && j + e < l ? fmaf(beta, value<PL>(pre, e), alpha * v[e]) : 0.f;
    if (i < k && j < x_cols) put8<PL>(x + b * x_batch + (int64_t)i * x_pitch, j, v);
  }
  __device__ __forceinline__ bool columns(bool) const { return true; }
  __device__ __forceinline__ void col8(int b, int i, int j, const float (&v)[8]) const {
    if (j < l && i < t_cols) put8<PL>(xt + b * t_batch + (int64_t)j * t_pitch, i, v);
  }
};

// The last step's: O, or the weights that it updates.
template <int PL>
struct LastStore {
  static constexpr bool kSymmetric = false;
  static constexpr bool kSplit = false;
  void* out[kBatch];
  const half_t* x;
  int dtype, tall, update;
  int64_t stride;
  int k, l, x_pitch, x_cols;
  int64_t x_batch;
  float alpha, beta, keep, rate;
  using Pre = Halves<PL>;
  __device__ __forceinline__ Pre fetch(int b, int i, int j) const {
    Pre r{};
    if (i < k && j < x_cols) r = get8<PL>(x + b * x_batch + (int64_t)i * x_pitch, j);
    return r;
  }
  __device__ __forceinline__ void emit(int b, int r, int c, int count, const float (&v)[8]) const {
    if (count <= 0) return;
    const int64_t o = r * stride + c;
    float w[8];
    if (update) load8(out[b], o, dtype, count, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = update ? fmaf(-rate, v[e], keep * w[e]) : v[e];
    store8(out[b], o, dtype, count, w);
  }
  __device__ __forceinline__ void row8(int b, int i, int j, float (&v)[8], const Pre& pre) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf(beta, value<PL>(pre, e), alpha * v[e]);
    if (!tall) emit(b, i, j, i < k ? l - j : 0, v);
  }
  __device__ __forceinline__ bool columns(bool) const { return tall; }
  __device__ __forceinline__ void col8(int b, int i, int j, const float (&v)[8]) const {
    emit(b, j, i, j < l ? k - i : 0, v);
  }
};

// T x T tiles of WM x WN waves, kB x kB matrix products, S stages of 128 bytes a row in LDS.
// Bound by LDS, written at 64 and read at 128 bytes a clock: a stage of one tile on an idle chip
// takes 0.27, 0.58, 0.74 and 1.12 us at T = 64, 128, 192 and 256, of which the matrix cores need
// 0.05, 0.21, 0.48 and 0.85; on a full chip by power.  B X of 4096 x 4096 in half precision: 122
// us, 1130 TFLOP/s.
template <int T, int WM, int WN, int S, int kB, int PL, class Store>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(Operands o, Store store) {
  constexpr int kWaves = WM * WN;
  constexpr int kRowBytes = 128;
  constexpr int kStage = 2 * T * kRowBytes;
  constexpr int kGroup = 1024 / kRowBytes;           // rows of a wave's load
  constexpr int kLoads = 2 * T / kGroup / kWaves;    // loads a wave and stage
  constexpr int BM = T / WM / kB, BN = T / WN / kB;  // kB x kB blocks of a wave
  constexpr int kK = kB / 16;                        // products of 32 float16 along the rows
  constexpr int kCols = BN * kB;
  constexpr int kRegs = kB * kB / 64;
  typedef float acc_t __attribute__((ext_vector_type(kRegs)));
  constexpr int kPitch = kCols + 4;       // floats a row where the sums pass through LDS
  constexpr int kPass = 32 * kPitch * 4;  // bytes a wave needs there: 32 rows at a time
  constexpr int kLds = S * kStage > kWaves * kPass ? S * kStage : kWaves * kPass;
  static_assert(T % (kGroup * kWaves) == 0 && BM * kB % 32 == 0 && 32 * kCols / 8 % 64 == 0,
                "tile shape");
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Workgroups go round the eight XCDs in turn; each XCD is given tiles that lie next to each
  // other, so that its L2 holds the rows they share.
  int x = blockIdx.x;
  {
    const int per = o.tiles >> 3, more = o.tiles & 7, xcd = x & 7;
    x = xcd * per + min(xcd, more) + (x >> 3);
  }
  const int one = Store::kSymmetric ? o.tiles_p * (o.tiles_p + 1) / 2 : o.tiles_p * o.tiles_q;
  const int b = x / one;  // matrix, or matrix of a part of the sums
  x -= b * one;
  int matrix = b, steps = o.steps;
  int64_t skip = 0;
  if constexpr (Store::kSplit) {
    const int part = b / store.nb, from = part * store.per;
    matrix = b - part * store.nb;
    steps = min(store.per, o.steps - from);
    skip = (int64_t)from * 64;
  }
  int ti, tj;
  if (Store::kSymmetric) {
    ti = (int)((sqrtf(8.f * x + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > x) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= x) ++ti;
    tj = x - ti * (ti + 1) / 2;
  } else {
    // down four tiles, then across
    const int band = x / (4 * o.tiles_q), first = band * 4;
    const int high = min(4, o.tiles_p - first);
    x -= first * o.tiles_q;
    tj = x / high;
    ti = first + x - tj * high;
  }
  const int i0 = ti * T, j0 = tj * T;

  // A wave's load fills 1024 bytes, rows one after the other.  The 16-byte pieces of a row are
  // permuted by its number so that the rows that a wave reads a piece of at a time lie in
  // different banks.  Rows past the operand's last are copies of it, whose sums are not stored.
  auto permuted = [](int piece, int row) {
    return piece ^ ((kB == 16 ? row : row >> 1) & 7);
  };
  const half_t* pbase = scalar_base(o.p + matrix * o.p_batch + skip + (int64_t)i0 * o.p_pitch);
  const half_t* qbase = scalar_base(o.q + matrix * o.q_batch + skip + (int64_t)j0 * o.q_pitch);
  uint32_t off[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const bool second = q >= kLoads / 2;  // P's rows, then Q's
    const int row = (q % (kLoads / 2) * kWaves + wave) * kGroup + lane / (64 / kGroup);
    const int last = (second ? o.q_rows - j0 : o.p_rows - i0) - 1;
    const int pitch = second ? o.q_pitch : o.p_pitch;
    off[q] = (uint32_t)min(row, last) * (uint32_t)(pitch * 2) +
             permuted(lane % (64 / kGroup), row) * 16;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  uint32_t to = lds0 + wave * 1024;  // where the next stage's loads go
  auto load_some = [&](int from, int upto) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      if (q >= from && q < upto)
        load_lds16(q < kLoads / 2 ? pbase : qbase, off[q],
                   __builtin_amdgcn_readfirstlane(to + q * kWaves * 1024));
  };
  auto load_next = [&]() {
    pbase += kRowBytes / 2;
    qbase += kRowBytes / 2;
    to += kStage;
    if (to >= lds0 + S * kStage) to -= S * kStage;
  };

  acc_t acc[BM][BN];
#pragma unroll
  for (int m = 0; m < BM; ++m)
#pragma unroll
    for (int n = 0; n < BN; ++n)
#pragma unroll
      for (int e = 0; e < kRegs; ++e) acc[m][n][e] = 0.f;

  const int wi = (wave / WN) * (T / WM), wj = (wave % WN) * (T / WN);
  constexpr int kHalves = 2;  // 32 float16 of a row each
  const char* frag[kHalves * kK];
#pragma unroll
  for (int h = 0; h < kHalves * kK; ++h) {
    const int row = lane & (kB - 1);
    frag[h] = lds + row * kRowBytes + permuted(h * (4 / kK) + lane / kB, row) * 16;
  }
  auto read = [&](int stage, int h, int row, f16x8& f) {
    f = *reinterpret_cast<const f16x8*>(frag[h] + stage * kStage + row * kRowBytes);
  };
  // A run of products (fp, fq), row by row of blocks; between them, what is needed later is
  // fetched a little at a time, so that the wave does not stand behind its own requests: the
  // reads of half h of a stage to (np, nq), and loads from .. upto of a stage in the making.
  auto run = [&](const f16x8(&fp)[BM * kK], const f16x8(&fq)[BN * kK], bool reads, int stage, int h,
                 f16x8(&np)[BM * kK], f16x8(&nq)[BN * kK], bool loads, int from, int upto) {
#pragma unroll
    for (int m = 0; m < BM; ++m) {
      if (reads) {
        constexpr int R = (BM + BN) * kK;
#pragma unroll
        for (int r = m * R / BM; r < (m + 1) * R / BM; ++r) {
          if (r < BN * kK)
            read(stage, h * kK + r % kK, T + wj + r / kK * kB, nq[r < BN * kK ? r : 0]);
          else
            read(stage, h * kK + r % kK, wi + (r / kK - BN) * kB, np[r < BN * kK ? 0 : r - BN * kK]);
        }
      }
      if (loads) load_some(from + m * (upto - from) / BM, from + (m + 1) * (upto - from) / BM);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < kK; ++x)
#pragma unroll
        for (int n = 0; n < BN; ++n) {
          if constexpr (kB == 16)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[m], fq[n], acc[m][n], 0, 0, 0);
          else
            acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[m * kK + x], fq[n * kK + x],
                                                               acc[m][n], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Stage s is in LDS once at most the loads of the S - 2 after it are outstanding.  This wave's
  // reads are done, and after the barrier all waves': the stage read last may be refilled.
  auto arrive = [&](int s) {
    __builtin_amdgcn_sched_barrier(0);
    wait_reads();
    if (s + S - 1 <= steps)
      wait_tile<(S - 2) * kLoads>();
    else
      wait_tile<0>();
    workgroup_barrier();
  };
  // The last reads, of a stage past the last, are of no use and do no harm.
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < steps) {
      load_some(0, kLoads);
      load_next();
    }
  f16x8 p0[BM * kK], q0[BN * kK], p1[BM * kK], q1[BN * kK], q2[BN * kK];
  arrive(0);
  bool more = S - 1 < steps;  // whether there is a stage to load during this step
  int stage = 0;
#pragma unroll
  for (int m = 0; m < BM * kK; ++m) read(0, m % kK, wi + m / kK * kB, p0[m]);
#pragma unroll
  for (int n = 0; n < BN * kK; ++n) read(0, n % kK, T + wj + n / kK * kB, q0[n]);
  // Loads are issued between the products of a step's runs; with two stages, which leave them
  // one step to arrive in, all at once.
  constexpr int kRuns = PL == 2 ? 3 : kHalves;
  constexpr int kPart = S == 2 ? kLoads : kLoads / kRuns;
  auto begin = [&]() {
    if (S == 2 && more) load_some(0, kLoads);
  };
  auto next_stage = [&](int s) {
    if (more) load_next();
    arrive(s + 1);
    more = s + S < steps;
    stage = stage + 1 == S ? 0 : stage + 1;
    begin();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto part = [&](int r) { return S == 2 ? 0 : r == kRuns ? kLoads : r * kPart; };
  begin();
  if constexpr (PL == 1) {
    if (S > 2 && more) load_some(0, part(1));
    for (int s = 0; s < steps; ++s) {
      wait_reads();
      run(p0, q0, true, stage, kHalves - 1, p1, q1, more, part(1), part(2));
      next_stage(s);
      run(p1, q1, true, stage, 0, p0, q0, more, part(0), part(1));
    }
  } else {
    if (S > 2 && more) load_some(0, part(1));
    // q: the first halves of Q of this step, nq those of the next
    auto step = [&](int s, const f16x8(&q)[BN * kK], f16x8(&nq)[BN * kK]) {
      wait_reads();
      run(p0, q, true, stage, kHalves - 1, p1, q1, more, part(1), part(2));
      wait_reads();
      run(p0, q1, false, 0, 0, p1, q1, more, part(2), part(3));
      next_stage(s);
      run(p1, q, true, stage, 0, p0, nq, more, part(0), part(1));
    };
    for (int s = 0; s < steps; s += 2) {
      step(s, q0, q2);
      if (s + 1 < steps) step(s + 1, q2, q0);
    }
  }
  wait_reads();
  __builtin_amdgcn_sched_barrier(0);

  // The sums pass through the wave's own part of LDS, 32 rows at a time, so that rows and
  // columns of the result leave in 16-byte pieces.
  float* pass = reinterpret_cast<float*>(lds + wave * kPass);
  const bool columns = store.columns(Store::kSymmetric && ti == tj);
  constexpr int kUnits = 32 * kCols / 8 / 64;
  constexpr int kPasses = BM * kB / 32;
  typename Store::Pre pre[kPasses][kUnits];
#pragma unroll
  for (int m = 0; m < kPasses; ++m)
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at_u = u * 64 + lane;
      pre[m][u] = store.fetch(b, i0 + wi + m * 32 + at_u / (kCols / 8),
                              j0 + wj + at_u % (kCols / 8) * 8);
    }
#pragma unroll
  for (int m = 0; m < kPasses; ++m) {
    const int i = i0 + wi + m * 32, j = j0 + wj;
#pragma unroll
    for (int n = 0; n < BN; ++n) {
      if constexpr (kB == 16) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          pass[(r / 4 * 16 + (lane >> 4) * 4 + r % 4) * kPitch + n * 16 + (lane & 15)] =
              acc[m * 2 + r / 4][n][r % 4];
      } else {
#pragma unroll
        for (int r = 0; r < kRegs; ++r)
          pass[(r / 4 * 8 + (lane >> 5) * 4 + r % 4) * kPitch + n * 32 + (lane & 31)] =
              acc[m][n][r];
      }
    }
    wave_order();
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int at_u = u * 64 + lane, r = at_u / (kCols / 8), c = at_u % (kCols / 8) * 8;
      float* q = pass + r * kPitch + c;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(q);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(q + 4);
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      store.row8(b, i + r, j + c, v, pre[m][u]);
      if (columns) {
        *reinterpret_cast<f32x4*>(q) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(q + 4) = f32x4{v[4], v[5], v[6], v[7]};
      }
    }
    wave_order();
    if (columns) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int at_u = u * 64 + lane, c = at_u >> 2, r = (at_u & 3) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = pass[(r + e) * kPitch + c];
        store.col8(b, i + r, j + c, v);
      }
      wave_order();
    }
  }
}

// ------------------------------------------------------------ a short side
// Where k is at most 64 the products of a step are too small for the chip, and their launches
// are most of the time.  There the steps go over the Gram matrix alone: with P = a + b A + c A A,
// X becomes P X, so A becomes P A P and, of all steps, O = P_last .. P_1 X_0 = Q X_0.  Three
// launches: G = U U' (||U||_F^2 is its trace), Q in one workgroup's LDS, Q U.  A rounding of A in
// the directions that X_0 hardly has grows by a^2 a step, where the products of X keep A = X X'
// whole; so all of this is in 64 bits, and a^(2 steps) is bounded (kGramGrowth).  Against the
// tiles, us: 32 x 200 fp32 74 -> 22, 64 x 2000 96 -> 65.
constexpr int kGram = 64;
constexpr double kGramGrowth = 1e9;  // times 2^-53: 1e-7 of a step's polynomial
constexpr int kGramBlocks = 32;      // most workgroups that sum a Gram matrix

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Columns j0 .. j0 + 63 of U (of its transpose, where U is tall) into LDS, zeros past its edges:
// row r of column j0 + c at tile[r][c], or at tile[c][r] if `kByColumn` is set.  The momentum is
// updated on the way if `first` is.
template <int KP, bool kByColumn, class Tile>
__device__ __forceinline__ void load_block(const Source& s, int b, int j0, bool first,
                                           Tile& tile) {
  const bool tall = s.m > s.n;
  const int k = tall ? s.n : s.m, l = tall ? s.m : s.n;
  const void* g = s.g[b];
  void* mom = s.mom[b];
#pragma unroll
  for (int q = 0; q < KP * 64 / 256; ++q) {
    const int x = q * 256 + threadIdx.x;
    const int r = tall ? x % KP : x / 64, c = tall ? x / KP : x % 64;
    const int j = j0 + c;
    float u = 0.f;
    if (r < k && j < l) {
      const int row = tall ? j : r, col = tall ? r : j;
      u = load1(g, row * s.g_stride + col, s.g_dtype);
      if (mom) {
        const int64_t at_m = row * s.m_stride + col;
        float v = load1(mom, at_m, s.m_dtype);
        if (first) {
          v = fmaf(s.mu, v, u);
          if (s.m_dtype != 0) v = widen(narrow(v, s.m_dtype), s.m_dtype);
          store1(mom, at_m, s.m_dtype, v);
        }
        u = s.nesterov ? fmaf(s.mu, v, u) : v;
      }
    }
    tile[kByColumn ? c : r][kByColumn ? r : c] = u;
  }
}

// A 16 x 16 block of lhs rhs' in 64 bits, sums over `len` columns: lane n reads row n % 16 of both
// and gets rows n / 16 + 4 r of column n % 16 in element r.
template <int len, class L, class R>
__device__ __forceinline__ f64x4 block64(const L* lhs, int lhs_pitch, const R* rhs, int rhs_pitch,
                                         f64x4 acc) {
  const int lane = threadIdx.x & 63;
  const L* p = lhs + (lane & 15) * lhs_pitch + (lane >> 4);
  const R* q = rhs + (lane & 15) * rhs_pitch + (lane >> 4);
#pragma unroll
  for (int t = 0; t < len; t += 4)
    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)p[t], (double)q[t], acc, 0, 0, 0);
  return acc;
}

// Block x on or below the diagonal, row by row of blocks.
__device__ __forceinline__ void below(int x, int& ti, int& tj) {
  ti = 0;
  while ((ti + 1) * (ti + 2) / 2 <= x) ++ti;
  tj = x - ti * (ti + 1) / 2;
}

template <int KP>
__global__ __launch_bounds__(256) void gram_kernel(Source s, double* __restrict__ partial) {
  __shared__ float tile[KP][65];
  constexpr int kBlocks = KP / 16 * (KP / 16 + 1) / 2, kEach = (kBlocks + 3) / 4;
  const int l = max(s.m, s.n);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f64x4 acc[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) acc[e] = f64x4{0.0, 0.0, 0.0, 0.0};
  for (int j0 = blockIdx.x * 64; j0 < l; j0 += gridDim.x * 64) {
    __syncthreads();
    load_block<KP, false>(s, blockIdx.y, j0, true, tile);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      int ti, tj;
      below(min(wave + 4 * e, kBlocks - 1), ti, tj);
      acc[e] = block64<64>(&tile[ti * 16][0], 65, &tile[tj * 16][0], 65, acc[e]);
    }
  }
  double* out = partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * KP * KP;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    int ti, tj;
    below(min(wave + 4 * e, kBlocks - 1), ti, tj);
    if (wave + 4 * e < kBlocks) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ti * 16 + (lane >> 4) + 4 * r, j = tj * 16 + (lane & 15);
        if (i >= j) {
          out[i * KP + j] = acc[e][r];
          out[j * KP + i] = acc[e][r];
        }
      }
    }
  }
}

// Q / (||U||_F + eps) of one matrix.  The operands are symmetric and commute; a wave takes a
// 16 x 16 block on or below the diagonal of each product and writes it to both sides.
template <int KP>
__global__ __launch_bounds__(64 * (KP / 16) * (KP / 16)) void polynomial_kernel(
    const double* __restrict__ partial, int blocks, double* __restrict__ out, int steps, double a,
    double b, double c, double eps) {
  constexpr int R = KP / 16, kThreads = 64 * R * R, kPitch = KP + 1;
  __shared__ double A[KP * kPitch], P[KP * kPitch], Q[KP * kPitch];
  __shared__ double trace;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int ti, tj;
  below(wave, ti, tj);
  const bool active = ti < R;
  {
    const int x = 4 * threadIdx.x;  // KP * KP elements, four a thread
    const f64x4* g = reinterpret_cast<const f64x4*>(partial + (int64_t)blockIdx.x * blocks * KP *
                                                                  KP + x);
    f64x4 v{0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
    for (int i = 0; i < blocks; ++i) v += g[(int64_t)i * (KP * KP / 4)];
#pragma unroll
    for (int e = 0; e < 4; ++e) A[x / KP * kPitch + x % KP + e] = v[e];
  }
  static_assert(4 * kThreads == KP * KP, "four elements a thread");
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int i = 0; i < KP; ++i) v += A[i * kPitch + i];
    trace = v;
  }
  __syncthreads();
  const double f = sqrt(trace) + eps;
  const double inv = f > 0.0 ? 1.0 / f : (f == 0.0 ? 0.0 : NAN);
  for (int x = threadIdx.x; x < KP * KP; x += kThreads) {
    const int at = x / KP * kPitch + x % KP;
    A[at] *= inv * inv;
    Q[at] = x / KP == x % KP ? 1.0 : 0.0;
  }
  __syncthreads();
  auto product = [&](const double* p, const double* q) {
    const f64x4 zero{0.0, 0.0, 0.0, 0.0};
    return active ? block64<KP>(p + ti * 16 * kPitch, kPitch, q + tj * 16 * kPitch, kPitch, zero)
                  : zero;
  };
  auto put = [&](double* to, const f64x4& v) {
    if (active) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ti * 16 + (lane >> 4) + 4 * r, j = tj * 16 + (lane & 15);
        if (i >= j) {
          to[i * kPitch + j] = v[r];
          to[j * kPitch + i] = v[r];
        }
      }
    }
    __syncthreads();
  };
  for (int s = 0; s < steps; ++s) {
    f64x4 v = product(A, A);
    if (active) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ti * 16 + (lane >> 4) + 4 * r, j = tj * 16 + (lane & 15);
        v[r] = c * v[r] + b * A[i * kPitch + j] + (i == j ? a : 0.0);
      }
    }
    put(P, v);
    if (s == 0) {
      for (int x = threadIdx.x; x < KP * kPitch; x += kThreads) Q[x] = P[x];
      __syncthreads();
    } else {
      v = product(P, Q);
      __syncthreads();
      put(Q, v);
    }
    if (s + 1 == steps) break;
    v = product(P, A);
    __syncthreads();
    put(A, v);
    v = product(A, P);
    __syncthreads();
    put(A, v);
  }
  double* o = out + (int64_t)blockIdx.x * KP * KP;
  for (int x = threadIdx.x; x < KP * KP; x += kThreads)
    o[x] = Q[x / KP * kPitch + x % KP] * inv;
}

// O = Q U for 64 columns of U (rows, where it is tall), or the weights that it updates.
struct ApplyStore {
  void* out[kBatch];
  int dtype, update;
  int64_t stride;
  float keep, rate;
};

template <int KP>
__global__ __launch_bounds__(256) void apply_kernel(Source s, const double* __restrict__ poly,
                                                    ApplyStore store) {
  __shared__ float tile[64][KP + 1];  // U's columns as rows
  __shared__ double q[KP * (KP + 1)];
  const bool tall = s.m > s.n;
  const int k = min(s.m, s.n), l = max(s.m, s.n), b = blockIdx.y, j0 = blockIdx.x * 64;
  load_block<KP, true>(s, b, j0, false, tile);
  for (int x = threadIdx.x; x < KP * KP; x += 256)
    q[x / KP * (KP + 1) + x % KP] = poly[(int64_t)b * KP * KP + x];
  __syncthreads();  // the result may lie where U did
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int x = 0; x < KP / 16; ++x) {
    // Q is symmetric: either factor may give the rows.  Neighbouring lanes take neighbouring
    // elements of the result's rows.
    const f64x4 zero{0.0, 0.0, 0.0, 0.0};
    const double* qr = q + x * 16 * (KP + 1);
    const float* ur = &tile[wave * 16][0];
    const f64x4 acc = tall ? block64<KP>(ur, KP + 1, qr, KP + 1, zero)
                           : block64<KP>(qr, KP + 1, ur, KP + 1, zero);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = (lane >> 4) + 4 * r, col = lane & 15;
      const int i = x * 16 + (tall ? col : row), j = j0 + wave * 16 + (tall ? row : col);
      if (i < k && j < l) {
        const int64_t o = tall ? j * store.stride + i : i * store.stride + j;
        float v = (float)acc[r];
        if (store.update)
          v = fmaf(-store.rate, v, store.keep * load1(store.out[b], o, store.dtype));
        store1(store.out[b], o, store.dtype, v);
      }
    }
  }
}

// ----------------------------------------------------------------- host side
struct Plan {
  int64_t k, l;
  int kp, lp;                 // rows of length k and l in float16, padded, both halves
  int kcols, lcols;           // the elements they hold, padded
  int64_t x, xt, a;           // float16 of X, X' and A (or B) a matrix
  size_t partials;            // bytes
  int per;                    // matrices a launch
  int gram;                   // k padded to 16, 32 or 64 where it is that short, else 0
  int gram_blocks;
  bool split;                 // whether X X' may be summed in parts
  size_t bytes;
};

int make_plan(int64_t m, int64_t n, int64_t count, int precision, Plan* p) {
  if (m < 0 || n < 0 || count < 0)
    return nl2k::fail(NL2K_ERR_SHAPE, "need m, n, count >= 0, got m=%lld n=%lld count=%lld",
                      (long long)m, (long long)n, (long long)count);
  if (precision != 1 && precision != 2)
    return nl2k::fail(NL2K_ERR_VALUE, "precision must be 1 (half) or 2 (full), got %d", precision);
  // rows and columns are counted in 32 bits, tiles in a launch's 16 bits of y
  if (m > 1 << 21 || n > 1 << 21 || std::min(m, n) > 1 << 16)
    return nl2k::fail(NL2K_ERR_OVERFLOW,
                      "m and n must be at most 2^21 and one of them 2^16, got %lld x %lld",
                      (long long)m, (long long)n);
  p->k = std::min(m, n);
  p->l = std::max(m, n);
  const int unit = kStep / precision;  // elements of a stage
  p->kcols = (int)(nl2k::ceil_div(p->k, (int64_t)unit) * unit);
  p->lcols = (int)(nl2k::ceil_div(p->l, (int64_t)unit) * unit);
  p->kp = p->kcols * precision;
  p->lp = p->lcols * precision;
  p->x = p->k * p->lp;
  p->xt = p->l * p->kp;
  p->a = p->k * p->kp;
  const size_t one = 2 * (size_t)(p->x + 2 * p->xt + 2 * p->a);
  p->per = (int)std::max<int64_t>(
      1, std::min<int64_t>({count, kBatch, (int64_t)(kMaxBatchBytes / std::max<size_t>(one, 1))}));
  p->partials = (size_t)p->per * kPartials * sizeof(double);
  p->bytes = p->partials + p->per * one;
  const int64_t t = nl2k::ceil_div(p->k, (int64_t)64);
  p->split = t * (t + 1) <= kSplitTiles && p->lp >= 8 * kStep;  // two parts of four stages
  if (p->split) p->bytes += (size_t)kSplitTiles * kSplitTile * sizeof(float);
  p->gram = p->k > kGram ? 0 : p->k > 32 ? 64 : p->k > 16 ? 32 : 16;
  p->gram_blocks = (int)std::min<int64_t>(nl2k::ceil_div(std::max<int64_t>(p->l, 1), 64),
                                          kGramBlocks);
  if (p->gram) {  // the steps may ask for either way
    const size_t square = (size_t)p->gram * p->gram * sizeof(double);
    p->bytes = std::max(p->bytes, p->per * square * (p->gram_blocks + 1));
  }
  return NL2K_SUCCESS;
}

// Powers of two that take X, A and B to float16's range, from the largest
// singular values that the steps can meet.
struct Scales {
  float x, a, b;
};

int make_scales(int steps, float a, float b, float c, Scales* s) {
  if (!(std::fabs(a) < 1e3f && std::fabs(b) < 1e3f && std::fabs(c) < 1e3f))
    return nl2k::fail(NL2K_ERR_VALUE,
                      "coefficients must be finite and below 1000, got (%g, %g, %g)", (double)a,
                      (double)b, (double)c);
  double top = 1.0, top_x = 1.0, top_b = 0.0;
  for (int i = 0; i < steps; ++i) {
    double next = 0.0;
    constexpr int kGrid = 512;
    for (int g = 0; g <= kGrid; ++g) {
      const double v = top * g / kGrid, q = v * v;
      next = std::max(next, std::fabs(v * (a + q * (b + q * c))));
      top_b = std::max(top_b, std::fabs(q * (b + q * c)));
    }
    next *= 1.001;  // between the points of the grid
    if (!(next <= 4.0))
      return nl2k::fail(NL2K_ERR_VALUE,
                        "coefficients (%g, %g, %g) take a singular value in [0, 1] to %g in %d "
                        "steps, past 4", (double)a, (double)b, (double)c, next, i + 1);
    top = std::max(next, 1e-3);
    top_x = std::max(top_x, next);
  }
  // an eighth of room for rounding
  auto power = [](double most) {
    return (float)std::exp2(std::floor(std::log2(65504.0 * 0.875 / most)));
  };
  s->x = power(top_x);
  s->a = power(top_x * top_x);
  s->b = power(std::max(top_b, 1e-3));
  return NL2K_SUCCESS;
}

template <int T, int WM, int WN, int S, int kB, int PL, class Store>
int launch_tiles(Operands o, const Store& store, int nb, hipStream_t stream) {
  o.steps = o.row_bytes / 128;
  o.tiles_p = (int)nl2k::ceil_div(o.p_rows, T);
  o.tiles_q = (int)nl2k::ceil_div(o.q_rows, T);
  const int64_t tiles = (int64_t)nb * (Store::kSymmetric ? (int64_t)o.tiles_p * (o.tiles_p + 1) / 2
                                                         : (int64_t)o.tiles_p * o.tiles_q);
  if (tiles > nl2k::max_blocks(64 * WM * WN) || tiles > INT32_MAX)
    return nl2k::fail(NL2K_ERR_OVERFLOW, "product of %lld tiles is more than a launch has",
                      (long long)tiles);
  o.tiles = (int)tiles;
  hipLaunchKernelGGL((product_kernel<T, WM, WN, S, kB, PL, Store>), dim3((unsigned)tiles),
                     dim3(64 * WM * WN), 0, stream, o, store);
  return nl2k::check_launch("product_kernel");
}

// Tile shapes and what they were measured to take, in us: a product's fixed part, a stage of a
// tile alone on its CU, and a stage where all CUs hold `per_cu` of them.  Between those lies a
// round that is part full; full rounds of large tiles draw the chip's power limit.  More stages
// in LDS changed nothing (64 x 64: 3, 5 or 9), nor did 64 bytes a row in place of 128.
struct Shape {
  int tile, per_cu;
  double fixed, alone, full;
};
constexpr int kShapes = 4;
constexpr Shape kHalfShapes[kShapes] = {
    {256, 1, 9.0, 1.13, 1.80}, {192, 1, 8.0, 0.76, 1.31}, {128, 2, 7.0, 0.55, 1.18},
    {64, 3, 4.0, 0.29, 0.64}};
constexpr Shape kFullShapes[kShapes] = {  // in full precision 256 x 256 does not fit the registers
    {0, 0, 0.0, 0.0, 0.0}, {192, 1, 8.0, 0.91, 1.69}, {128, 2, 7.0, 0.63, 1.53},
    {64, 3, 4.0, 0.31, 0.77}};

// Tiles of a product of matrices p x q; on and below the diagonal where it is symmetric.
double tiles_of(int64_t p, int64_t q, int tile, bool symmetric, int nb) {
  const double tp = (double)nl2k::ceil_div(p, (int64_t)tile);
  const double tq = (double)nl2k::ceil_div(q, (int64_t)tile);
  return nb * (symmetric ? tp * (tp + 1) / 2 : tp * tq);
}

// Time of a stage in `rounds` of a shape over 256 CUs.
double stage_time(const Shape& s, double tiles) {
  const double rounds = tiles / (256 * s.per_cu), rest = rounds - std::floor(rounds);
  return std::floor(rounds) * s.full + (rest > 0.0 ? s.alone + (s.full - s.alone) * rest : 0.0);
}

// The shape that takes least, and its time.
int choose(const Shape (&shapes)[kShapes], const Operands& o, bool symmetric, int nb,
           double* time) {
  int best = -1;
  for (int c = 0; c < kShapes; ++c) {
    const Shape& s = shapes[c];
    if (s.tile == 0) continue;
    const double t = s.fixed + stage_time(s, tiles_of(o.p_rows, o.q_rows, s.tile, symmetric, nb)) *
                                   (o.row_bytes / 128);
    if (best < 0 || t < *time) best = c, *time = t;
  }
  return best;
}

template <int PL, class Store>
int launch_product(const Operands& o, const Store& store, int nb, hipStream_t stream) {
  double time;
  switch (choose(PL == 1 ? kHalfShapes : kFullShapes, o, Store::kSymmetric, nb, &time)) {
    case 0:
      if constexpr (PL == 1) return launch_tiles<256, 2, 4, 2, 16, PL>(o, store, nb, stream);
      break;
    case 1: return launch_tiles<192, 2, 4, 3, 16, PL>(o, store, nb, stream);
    case 2: return launch_tiles<128, 2, 2, 2, 32, PL>(o, store, nb, stream);
  }
  return launch_tiles<64, 2, 2, 3, 16, PL>(o, store, nb, stream);
}

// A symmetric product of few tiles and long rows: cut along the rows into parts whose sums a
// second launch adds, where that takes less.
constexpr double kSplitTime = 6.0;  // the second launch

int splits_of(const Shape (&shapes)[kShapes], const Operands& o, int nb) {
  double least;
  choose(shapes, o, true, nb, &least);
  const Shape& s = shapes[kShapes - 1];
  const int steps = o.row_bytes / 128;
  const double tiles = tiles_of(o.p_rows, o.q_rows, 64, true, nb);
  int best = 1;
  for (int parts = 2; parts <= 16 && parts * tiles <= kSplitTiles && 4 * parts <= steps;
       parts *= 2) {
    const double t =
        s.fixed + stage_time(s, tiles * parts) * nl2k::ceil_div(steps, parts) + kSplitTime;
    if (t < least) best = parts, least = t;
  }
  return best;
}

template <int PL>
int launch_gram(const Operands& o, const SymmetricStore<PL>& store, int nb, float* parts,
                hipStream_t stream) {
  const int splits = parts ? splits_of(PL == 1 ? kHalfShapes : kFullShapes, o, nb) : 1;
  if (splits == 1) return launch_product<PL>(o, store, nb, stream);
  const int t = (int)nl2k::ceil_div(o.p_rows, 64), tiles = t * (t + 1) / 2;
  const int per = (int)nl2k::ceil_div(o.row_bytes / 128, splits);
  const int count = (int)nl2k::ceil_div(o.row_bytes / 128, per);  // none of them empty
  const int st = launch_tiles<64, 2, 2, 3, 16, PL>(o, SplitStore{parts, nb, per, tiles},
                                                   nb * count, stream);
  if (st) return st;
  hipLaunchKernelGGL((sum_kernel<PL>), dim3(tiles, nb), dim3(256), 0, stream, parts, count, store);
  return nl2k::check_launch("sum_kernel");
}

struct Job {
  Source src;
  void* const* out;
  int out_dtype, update;
  int64_t out_stride;
  float keep, rate;
  int steps;
  float a, b, c, eps;
};

template <int PL>
int run_batch(const Job& job, const Plan& p, const Scales& sc, int first, int nb, void* workspace,
              hipStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  half_t* x = reinterpret_cast<half_t*>(static_cast<char*>(workspace) + p.partials);
  half_t* xt = x + (int64_t)p.per * p.x;
  half_t* xt2 = xt + (int64_t)p.per * p.xt;
  half_t* ga = xt2 + (int64_t)p.per * p.xt;
  half_t* gb = ga + (int64_t)p.per * p.a;
  float* parts = reinterpret_cast<float*>(gb + (int64_t)p.per * p.a);
  const bool tall = job.src.m > job.src.n;
  const int blocks = (int)std::min<int64_t>(
      nl2k::ceil_div((int64_t)job.src.m * nl2k::ceil_div(job.src.n, 8), 256), kPartials);
  hipLaunchKernelGGL(square_kernel, dim3(blocks, nb), dim3(256), 0, stream, job.src, partial);
  int st = nl2k::check_launch("square_kernel");
  if (st) return st;
  const dim3 tiles((unsigned)nl2k::ceil_div(job.src.n, 64), (unsigned)nl2k::ceil_div(job.src.m, 64),
                   nb);
  hipLaunchKernelGGL((scale_kernel<PL>), tiles, dim3(256), 0, stream, job.src, partial, blocks,
                     job.eps, sc.x, tall ? xt : x, tall ? p.kp : p.lp, tall ? p.kcols : p.lcols,
                     tall ? p.xt : p.x, tall ? x : xt, tall ? p.lp : p.kp,
                     tall ? p.lcols : p.kcols, tall ? p.x : p.xt);
  if ((st = nl2k::check_launch("scale_kernel"))) return st;

  const int k = (int)p.k, l = (int)p.l;
  for (int i = 0; i < job.steps; ++i) {
    const Operands xx{x, x, k, k, p.lp, p.lp, p.x, p.x, p.lp * 2};
    st = launch_gram<PL>(
        xx, SymmetricStore<PL>{ga, nullptr, k, p.kp, p.kcols, p.a, sc.a / (sc.x * sc.x), 0.f}, nb,
        p.split ? parts : nullptr, stream);
    if (st) return st;
    const Operands aa{ga, ga, k, k, p.kp, p.kp, p.a, p.a, p.kp * 2};
    st = launch_product<PL>(
        aa, SymmetricStore<PL>{gb, ga, k, p.kp, p.kcols, p.a, job.c * sc.b / (sc.a * sc.a),
                               job.b * sc.b / sc.a}, nb, stream);
    if (st) return st;
    const Operands bx{gb, xt, k, l, p.kp, p.kp, p.a, p.xt, p.kp * 2};
    if (i + 1 < job.steps) {
      st = launch_product<PL>(
          bx, StepStore<PL>{x, xt2, k, l, p.lp, p.kp, p.lcols, p.kcols, p.x, p.xt, 1.f / sc.b,
                            job.a}, nb, stream);
    } else {
      LastStore<PL> last{{}, x, job.out_dtype, tall, job.update, job.out_stride, k, l, p.lp,
                         p.lcols, p.x, 1.f / (sc.b * sc.x), job.a / sc.x, job.keep, job.rate};
      for (int q = 0; q < nb; ++q) last.out[q] = job.out[first + q];
      st = launch_product<PL>(bx, last, nb, stream);
    }
    if (st) return st;
    std::swap(xt, xt2);
  }
  return nl2k::succeed();
}

template <int KP>
int run_gram(const Job& job, const Plan& p, int first, int nb, void* workspace,
             hipStream_t stream) {
  double* partial = static_cast<double*>(workspace);
  double* poly = partial + (int64_t)p.per * p.gram_blocks * KP * KP;
  hipLaunchKernelGGL((gram_kernel<KP>), dim3(p.gram_blocks, nb), dim3(256), 0, stream, job.src,
                     partial);
  int st = nl2k::check_launch("gram_kernel");
  if (st) return st;
  hipLaunchKernelGGL((polynomial_kernel<KP>), dim3(nb), dim3(64 * (KP / 16) * (KP / 16)), 0,
                     stream, partial, p.gram_blocks, poly, job.steps, (double)job.a,
                     (double)job.b, (double)job.c, (double)job.eps);
  if ((st = nl2k::check_launch("polynomial_kernel"))) return st;
  ApplyStore store{{}, job.out_dtype, job.update, job.out_stride, job.keep, job.rate};
  for (int q = 0; q < nb; ++q) store.out[q] = job.out[first + q];
  hipLaunchKernelGGL((apply_kernel<KP>), dim3((unsigned)nl2k::ceil_div(p.l, (int64_t)64), nb),
                     dim3(256), 0, stream, job.src, poly, store);
  return nl2k::check_launch("apply_kernel");
}

int check_scalars(const char* what, int steps, float eps) {
  if (steps < 1 || steps > 64)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: steps must be from 1 to 64, got %d", what, steps);
  if (!(eps >= 0.f) || !(eps < INFINITY))
    return nl2k::fail(NL2K_ERR_VALUE, "%s: eps must be finite and at least 0, got %g", what,
                      (double)eps);
  return NL2K_SUCCESS;
}

int check_matrices(const char* what, const char* name, const void* const* p, int dtype,
                   int64_t stride, int64_t m, int64_t n, int64_t count) {
  if (dtype < 0 || dtype > 2)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: dtype of %s must be 0, 1 or 2, got %d", what, name,
                      dtype);
  if (m * n * count == 0) return NL2K_SUCCESS;
  if (m > 1 && stride < n)
    return nl2k::fail(NL2K_ERR_SHAPE, "%s: row stride of %s must be at least n, got %lld", what,
                      name, (long long)stride);
  if (!p) return nl2k::fail(NL2K_ERR_NULL, "%s: %s is NULL", what, name);
  for (int64_t i = 0; i < count; ++i) {
    if (!p[i]) return nl2k::fail(NL2K_ERR_NULL, "%s: %s[%lld] is NULL", what, name, (long long)i);
    if (reinterpret_cast<uintptr_t>(p[i]) % (dtype == 0 ? 4 : 2))
      return nl2k::fail(NL2K_ERR_ALIGN, "%s: %s[%lld] is not aligned to its elements", what, name,
                        (long long)i);
  }
  return NL2K_SUCCESS;
}

int run_all(const char* what, Job& job, const void* const* grads, void* const* momenta,
            int64_t m, int64_t n, int64_t count, int precision, void* workspace,
            size_t workspace_bytes, hipStream_t stream) {
  Plan p;
  int st = make_plan(m, n, count, precision, &p);
  if (st) return st;
  Scales sc;
  if ((st = make_scales(job.steps, job.a, job.b, job.c, &sc))) return st;
  if (m == 0 || n == 0 || count == 0) return nl2k::succeed();
  if (!workspace || workspace_bytes < p.bytes)
    return nl2k::fail(NL2K_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", what,
                      workspace_bytes, p.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: workspace must be aligned to 256 bytes", what);
  job.src.m = (int)m;
  job.src.n = (int)n;
  for (int64_t first = 0; first < count; first += p.per) {
    const int nb = (int)std::min<int64_t>(p.per, count - first);
    for (int q = 0; q < nb; ++q) {
      job.src.g[q] = grads[first + q];
      job.src.mom[q] = momenta ? momenta[first + q] : nullptr;
    }
    const double growth = std::pow(std::max(1.0, std::fabs((double)job.a)), 2.0 * job.steps);
    if (p.gram && growth <= kGramGrowth)
      st = p.gram == 16   ? run_gram<16>(job, p, (int)first, nb, workspace, stream)
           : p.gram == 32 ? run_gram<32>(job, p, (int)first, nb, workspace, stream)
                          : run_gram<64>(job, p, (int)first, nb, workspace, stream);
    else
      st = precision == 1 ? run_batch<1>(job, p, sc, (int)first, nb, workspace, stream)
                          : run_batch<2>(job, p, sc, (int)first, nb, workspace, stream);
    if (st) return st;
  }
  return nl2k::succeed();
}

}  // namespace

extern "C" size_t newton_schulz_workspace_bytes(int64_t m, int64_t n, int64_t count,
                                                int precision) {
  Plan p;
  return make_plan(m, n, count, precision, &p) ? 0 : p.bytes;
}

extern "C" int newton_schulz(const void* const* in, int in_dtype, int64_t in_row_stride,
                             void* const* out, int out_dtype, int64_t out_row_stride, int64_t m,
                             int64_t n, int64_t count, int steps, float a, float b, float c,
                             float eps, int precision, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
  const char* what = "newton_schulz";
  int st = check_scalars(what, steps, eps);
  if (!st && (m < 0 || n < 0 || count < 0)) {
    Plan p;
    st = make_plan(m, n, count, precision, &p);
  }
  if (!st) st = check_matrices(what, "in", in, in_dtype, in_row_stride, m, n, count);
  if (!st)
    st = check_matrices(what, "out", const_cast<const void* const*>(out), out_dtype,
                        out_row_stride, m, n, count);
  if (st) return st;
  Job job{};
  job.src.g_dtype = in_dtype;
  job.src.g_stride = in_row_stride;
  job.out = out;
  job.out_dtype = out_dtype;
  job.out_stride = out_row_stride;
  job.steps = steps;
  job.a = a;
  job.b = b;
  job.c = c;
  job.eps = eps;
  return run_all(what, job, in, nullptr, m, n, count, precision, workspace, workspace_bytes,
                 stream);
}

extern "C" int muon_update(void* const* weights, int weight_dtype, int64_t weight_row_stride,
                           const void* const* grads, int grad_dtype, int64_t grad_row_stride,
                           void* const* momenta, int momentum_dtype, int64_t momentum_row_stride,
                           int64_t m, int64_t n, int64_t count, float mu, int nesterov, float lr,
                           float weight_decay, float scale, int steps, float a, float b, float c,
                           float eps, int precision, void* workspace, size_t workspace_bytes,
                           hipStream_t stream) {
  const char* what = "muon_update";
  int st = check_scalars(what, steps, eps);
  if (!st && (m < 0 || n < 0 || count < 0)) {
    Plan p;
    st = make_plan(m, n, count, precision, &p);
  }
  if (!st)
    st = check_matrices(what, "weights", const_cast<const void* const*>(weights), weight_dtype,
                        weight_row_stride, m, n, count);
  if (!st) st = check_matrices(what, "grads", grads, grad_dtype, grad_row_stride, m, n, count);
  if (!st)
    st = check_matrices(what, "momenta", const_cast<const void* const*>(momenta), momentum_dtype,
                        momentum_row_stride, m, n, count);
  if (st) return st;
  const float scalars[] = {mu, lr, weight_decay, scale};
  for (float v : scalars)
    if (!(std::fabs(v) < INFINITY))
      return nl2k::fail(NL2K_ERR_VALUE, "%s: mu, lr, weight_decay and scale must be finite", what);
  Job job{};
  job.src.g_dtype = grad_dtype;
  job.src.g_stride = grad_row_stride;
  job.src.m_dtype = momentum_dtype;
  job.src.m_stride = momentum_row_stride;
  job.src.mu = mu;
  job.src.nesterov = nesterov;
  job.out = weights;
  job.out_dtype = weight_dtype;
  job.out_stride = weight_row_stride;
  job.update = 1;
  job.keep = 1.f - lr * weight_decay;
  job.rate = lr * scale;
  job.steps = steps;
  job.a = a;
  job.b = b;
  job.c = c;
  job.eps = eps;
  return run_all(what, job, grads, momenta, m, n, count, precision, workspace, workspace_bytes,
                 stream);
}

extern "C" const char* newton_schulz_last_error(void) { return nl2k::error_slot().text; }
