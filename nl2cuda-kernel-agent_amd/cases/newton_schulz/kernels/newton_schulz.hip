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

namespace {

using nl2k::f32x4;
using nl2k::u32x4;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half_t;

constexpr int kBatch = 32;        // matrices of one launch: their pointers are kernel arguments
constexpr int kPartials = 256;    // most workgroups that sum a matrix's squares
constexpr int kStep = 64;         // float16 of a row a tile step takes: 128 bytes
constexpr size_t kMaxBatchBytes = (size_t)4 << 30;

// ------------------------------------------------------------------ elements
__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  const unsigned short h = static_cast<const unsigned short*>(p)[i];
  if (dtype == 1) return __builtin_bit_cast(float, (uint32_t)h << 16);
  return (float)__builtin_bit_cast(half_t, h);
}

__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float v) {
  if (dtype == 0)
    static_cast<float*>(p)[i] = v;
  else if (dtype == 1)
    static_cast<unsigned short*>(p)[i] = __builtin_bit_cast(unsigned short, (__bf16)v);
  else
    static_cast<half_t*>(p)[i] = (half_t)v;
}

// Where element t of an operand row lies, in float16 (the second half 32 on).
template <int PL>
__device__ __forceinline__ int64_t at(int t) {
  return PL == 1 ? t : (int64_t)(t >> 5) * 64 + (t & 31);
}

template <int PL>
__device__ __forceinline__ void put(half_t* row, int t, float v) {
  const half_t hi = (half_t)v;
  half_t* p = row + at<PL>(t);
  p[0] = hi;
  if (PL == 2) p[32] = (half_t)(v - (float)hi);
}

template <int PL>
__device__ __forceinline__ float get(const half_t* row, int t) {
  const half_t* p = row + at<PL>(t);
  return PL == 2 ? (float)p[0] + (float)p[32] : (float)p[0];
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

// U's element from G and the momentum after its update.
__device__ __forceinline__ float update_of(const Source& s, float g, float mom) {
  return s.nesterov ? fmaf(s.mu, mom, g) : mom;
}

// Momentum and the sum of U's squares: a partial sum in 64 bits a workgroup.
__global__ __launch_bounds__(256) void square_kernel(Source s, double* __restrict__ partial) {
  __shared__ double red[4];
  const int b = blockIdx.y;
  const void* g = s.g[b];
  void* mom = s.mom[b];
  double sum = 0.0;
  for (int i = blockIdx.x; i < s.m; i += gridDim.x)
    for (int j = threadIdx.x; j < s.n; j += 256) {
      float u = load_elem(g, i * s.g_stride + j, s.g_dtype);
      if (mom) {
        const int64_t at_m = i * s.m_stride + j;
        const float x = fmaf(s.mu, load_elem(mom, at_m, s.m_dtype), u);
        store_elem(mom, at_m, s.m_dtype, x);
        // the momentum as it is kept, so that U is what a reader of it would form
        u = update_of(s, u, load_elem(mom, at_m, s.m_dtype));
      }
      sum += (double)u * u;
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
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int b = blockIdx.z;
  double q = (int)threadIdx.x < blocks ? partial[(int64_t)b * kPartials + threadIdx.x] : 0.0;
  q = nl2k::wave_sum(q);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = q;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const double f = norm + (double)eps;
  // 0 / 0 is an update of zeros; sx / f may pass 32 bits where the elements are small
  const double scale = f > 0.0 ? sx / f : (f == 0.0 ? 0.0 : NAN);
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
#pragma unroll 4
  for (int r = r0; r < 64; r += 4) {
    const int i = i0 + r, j = j0 + c;
    float u = 0.f;
    if (i < s.m && j < s.n) {
      u = load_elem(s.g[b], i * s.g_stride + j, s.g_dtype);
      if (s.mom[b]) u = update_of(s, u, load_elem(s.mom[b], i * s.m_stride + j, s.m_dtype));
      u = (float)(u * scale);
    }
    tile[r][c] = u;
    // rows: [m, n] padded along n to rows_len, cols: [n, m] along m to cols_len
    if (i < s.m && j < rows_len) put<PL>(rows + b * rows_batch + (int64_t)i * rows_pitch, j, u);
  }
  __syncthreads();
#pragma unroll 4
  for (int r = r0; r < 64; r += 4) {
    const int j = j0 + r, i = i0 + c;
    if (j < s.n && i < cols_len) put<PL>(cols + b * cols_batch + (int64_t)j * cols_pitch, i, tile[c][r]);
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
  int steps;                 // tile steps along a row
};

__device__ __forceinline__ void load_lds16(const half_t* g, char* l) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void*)g,
      (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// A symmetric result [n, n], both triangles from the tiles on and below the
// diagonal: v = alpha acc + beta D.
template <int PL>
struct SymmetricStore {
  static constexpr bool kSymmetric = true;
  half_t* c;
  const half_t* d;
  int n, pitch, cols;  // cols: n padded to a tile step
  int64_t batch;
  float alpha, beta;
  __device__ __forceinline__ void operator()(int b, int i, int j, float acc, bool diagonal) const {
    float v = alpha * acc;
    const bool in = i < n && j < n;
    if (in && d) v = fmaf(beta, get<PL>(d + b * batch + (int64_t)i * pitch, j), v);
    if (!in) v = 0.f;
    if (i < n && j < cols) put<PL>(c + b * batch + (int64_t)i * pitch, j, v);
    if (!diagonal && j < n && i < cols) put<PL>(c + b * batch + (int64_t)j * pitch, i, v);
  }
};

// X = alpha acc + beta X, as [k, l] in place and as [l, k].
template <int PL>
struct StepStore {
  static constexpr bool kSymmetric = false;
  half_t* x;
  half_t* xt;
  int k, l, x_pitch, t_pitch, x_cols, t_cols;
  int64_t x_batch, t_batch;
  float alpha, beta;
  __device__ __forceinline__ void operator()(int b, int i, int j, float acc, bool) const {
    const bool in = i < k && j < l;
    half_t* row = x + b * x_batch + (int64_t)i * x_pitch;
    const float v = in ? fmaf(beta, get<PL>(row, j), alpha * acc) : 0.f;
    if (i < k && j < x_cols) put<PL>(row, j, v);
    if (j < l && i < t_cols) put<PL>(xt + b * t_batch + (int64_t)j * t_pitch, i, v);
  }
};

// The last step's: O, or the weights that it updates.
template <int PL>
struct LastStore {
  static constexpr bool kSymmetric = false;
  void* out[kBatch];
  const half_t* x;
  int dtype, tall, update;
  int64_t stride;
  int k, l, x_pitch;
  int64_t x_batch;
  float alpha, beta, keep, rate;
  __device__ __forceinline__ void operator()(int b, int i, int j, float acc, bool) const {
    if (i >= k || j >= l) return;
    const float v =
        fmaf(beta, get<PL>(x + b * x_batch + (int64_t)i * x_pitch, j), alpha * acc);
    const int64_t o = tall ? j * stride + i : i * stride + j;
    store_elem(out[b], o, dtype,
               update ? fmaf(-rate, v, keep * load_elem(out[b], o, dtype)) : v);
  }
};

// T x T tiles, four waves of T/2 x T/2, two stages of a tile step in LDS.
template <int T, int PL, class Store>
__global__ __launch_bounds__(256) void product_kernel(Operands o, Store store) {
  constexpr int kRowBytes = kStep * 2;
  constexpr int kStage = 2 * T * kRowBytes;
  constexpr int kLoads = T / 32;   // 16-byte loads a thread and operand
  constexpr int W = T / 2 / 16;    // 16 x 16 blocks a wave, each way
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int ti, tj;
  if (Store::kSymmetric) {
    const int x = blockIdx.x;
    ti = (int)((sqrtf(8.f * x + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > x) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= x) ++ti;
    tj = x - ti * (ti + 1) / 2;
  } else {
    ti = blockIdx.x;
    tj = blockIdx.y;
  }
  const int b = blockIdx.z;
  const int i0 = ti * T, j0 = tj * T;

  // a wave's load fills eight rows of 128 bytes; the 16-byte pieces of a row are permuted by
  // its number so that the reads below meet no bank twice
  const int sub = lane >> 3, piece = (lane & 7) ^ sub;
  const half_t* src[2 * kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const int row = (q * 4 + wave) * 8 + sub;
    src[q] = o.p + b * o.p_batch + (int64_t)min(i0 + row, o.p_rows - 1) * o.p_pitch + piece * 8;
    src[kLoads + q] =
        o.q + b * o.q_batch + (int64_t)min(j0 + row, o.q_rows - 1) * o.q_pitch + piece * 8;
  }
  auto load = [&](int step, int stage) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      char* at_row = lds + stage * kStage + (q * 4 + wave) * 1024;
      load_lds16(src[q] + (int64_t)step * kStep, at_row);
      load_lds16(src[kLoads + q] + (int64_t)step * kStep, at_row + T * kRowBytes);
    }
  };

  f32x4 acc[W][W];
#pragma unroll
  for (int x = 0; x < W; ++x)
#pragma unroll
    for (int y = 0; y < W; ++y) acc[x][y] = nl2k::zero4();

  const int wi = (wave >> 1) * (T / 2), wj = (wave & 1) * (T / 2);
  const int frag_row = lane & 15;
  int frag[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    frag[h] = frag_row * kRowBytes + (((h * 4 + (lane >> 4)) ^ (lane & 7)) << 4);

  load(0, 0);
  for (int s = 0; s < o.steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tile is in LDS,
    __syncthreads();                     // then all of it is, and the other stage is free
    const char* pa = lds + (s & 1) * kStage + wi * kRowBytes;
    const char* qa = lds + (s & 1) * kStage + (T + wj) * kRowBytes;
    f16x8 fp[2][W], fq[2][W];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < W; ++x) {
        fp[h][x] = *reinterpret_cast<const f16x8*>(pa + x * 16 * kRowBytes + frag[h]);
        fq[h][x] = *reinterpret_cast<const f16x8*>(qa + x * 16 * kRowBytes + frag[h]);
      }
    if (s + 1 < o.steps) load(s + 1, (s + 1) & 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y) {
          if (PL == 1) {
            acc[x][y] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[h][x], fq[h][y], acc[x][y], 0, 0, 0);
          } else if (h == 0) {
            acc[x][y] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][x], fq[0][y], acc[x][y], 0, 0, 0);
          } else {
            acc[x][y] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[0][x], fq[1][y], acc[x][y], 0, 0, 0);
            acc[x][y] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[1][x], fq[0][y], acc[x][y], 0, 0, 0);
          }
        }
  }
#pragma unroll
  for (int x = 0; x < W; ++x)
#pragma unroll
    for (int y = 0; y < W; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        store(b, i0 + wi + x * 16 + (lane >> 4) * 4 + r, j0 + wj + y * 16 + frag_row,
              acc[x][y][r], Store::kSymmetric && ti == tj);
}

// ----------------------------------------------------------------- host side
struct Plan {
  int64_t k, l;
  int kp, lp;                 // rows of length k and l in float16, padded, both halves
  int kcols, lcols;           // the elements they hold, padded
  int64_t x, xt, a;           // float16 of X, X' and A (or B) a matrix
  size_t partials;            // bytes
  int per;                    // matrices a launch
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
  const int unit = kStep / precision;  // elements of a tile step
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
  return NL2K_SUCCESS;
}

// Powers of two that take X, A and B to float16's range, from the largest
// singular values that the steps can meet.
struct Scales {
  float x, a, b;
};

int make_scales(int steps, float a, float b, float c, Scales* s) {
  if (!(std::fabs(a) < 1e3f && std::fabs(b) < 1e3f && std::fabs(c) < 1e3f))
    return nl2k::fail(NL2K_ERR_VALUE, "coefficients must be finite and below 1000, got (%g, %g, %g)",
                      (double)a, (double)b, (double)c);
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

template <int PL, class Store>
int launch_product(const Operands& o, const Store& store, int nb, hipStream_t stream) {
  auto go = [&](auto tag) {
    constexpr int T = decltype(tag)::value;
    const int64_t ti = nl2k::ceil_div(o.p_rows, T), tj = nl2k::ceil_div(o.q_rows, T);
    const dim3 grid = Store::kSymmetric ? dim3((unsigned)(ti * (ti + 1) / 2), 1, nb)
                                        : dim3((unsigned)ti, (unsigned)tj, nb);
    hipLaunchKernelGGL((product_kernel<T, PL, Store>), grid, dim3(256), 0, stream, o, store);
    return nl2k::check_launch("product_kernel");
  };
  const int64_t big = nl2k::ceil_div(o.p_rows, 128) * nl2k::ceil_div(o.q_rows, 128) * nb /
                      (Store::kSymmetric ? 2 : 1);
  if (big >= 256) return go(std::integral_constant<int, 128>{});
  return go(std::integral_constant<int, 64>{});
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
  const bool tall = job.src.m > job.src.n;
  const int blocks = (int)std::min<int64_t>(job.src.m, kPartials);
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
    const Operands xx{x, x, k, k, p.lp, p.lp, p.x, p.x, p.lp / kStep};
    st = launch_product<PL>(
        xx, SymmetricStore<PL>{ga, nullptr, k, p.kp, p.kcols, p.a, sc.a / (sc.x * sc.x), 0.f}, nb,
        stream);
    if (st) return st;
    const Operands aa{ga, ga, k, k, p.kp, p.kp, p.a, p.a, p.kp / kStep};
    st = launch_product<PL>(
        aa, SymmetricStore<PL>{gb, ga, k, p.kp, p.kcols, p.a, job.c * sc.b / (sc.a * sc.a),
                               job.b * sc.b / sc.a}, nb, stream);
    if (st) return st;
    const Operands bx{gb, xt, k, l, p.kp, p.kp, p.a, p.xt, p.kp / kStep};
    if (i + 1 < job.steps) {
      st = launch_product<PL>(
          bx, StepStore<PL>{x, xt2, k, l, p.lp, p.kp, p.lcols, p.kcols, p.x, p.xt, 1.f / sc.b,
                            job.a}, nb, stream);
    } else {
      LastStore<PL> last{{}, x, job.out_dtype, tall, job.update, job.out_stride, k, l, p.lp, p.x,
                         1.f / (sc.b * sc.x), job.a / sc.x, job.keep, job.rate};
      for (int q = 0; q < nb; ++q) last.out[q] = job.out[first + q];
      st = launch_product<PL>(bx, last, nb, stream);
    }
    if (st) return st;
    std::swap(xt, xt2);
  }
  return nl2k::succeed();
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
