// Products of e4m3 matrices with a scale for each block of 128, for MI355X
// (gfx950).  C-ABI in include/block_matmul.h.
//
// The matrix instruction takes 16 rows of each operand and 128 numbers of k, a
// block: 32 a lane, lane l rows l % 16, k from 32 (l / 16) on.  b's rows are its
// first operand and a's its second, so that a lane's sums are of one row of a
// and of numbers next to each other in a row of the result.
//
// Scales that are powers of two the instruction applies itself.  32-bit ones
// are applied to a block's sums, in registers: sum += (sa sb) block.
//
// The 8-bit instruction adds eight products at a time in a narrow window: what
// lies 13 bits below the largest of the eight is dropped, and the result of
// numbers like a layer's is off by 1.5e-5 of its size (measured; 9.8e-9 with
// the 16-bit one).  That is a hundredth of what rounding to 16 bits costs, so
// 16-bit results are computed with it.  For 32-bit results the codes become
// bfloat16, which holds them exactly, and the 16-bit instruction, at half the
// rate, keeps every product whole.

#include "block_matmul.h"

#include "e4m3.h"
#include "lds_direct.h"

namespace {

using namespace nl2k::e4m3;
using namespace nl2k::lds;
using nl2k::f32x4;
using nl2k::u32x4;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How scales are applied: by the instruction, or afterwards, with those of b the same for 128
// rows or for one.
enum Mode { kHardware, kTiles, kRows };

struct Side {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t pitch;
  int64_t s_row, s_block;  // bytes between rows' (or tiles') and blocks' scales
  int32_t rows;
  int32_t shift;           // rows that share a scale: 1 << shift
};

struct Args {
  Side a, b;
  void* out;
  float* partial;  // sums of parts of k, [splits][M][N], or null
  int32_t K, steps;
  int32_t per;     // steps of a part
  int32_t tiles_a, tiles_b, tiles;
  int out_dtype;
};

// Lane group g's 32 numbers of a block of which `valid` count: the others 0.
__device__ __forceinline__ void cut(i32x8& f, int valid, int group) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = valid - 32 * group - 4 * i;
    f[i] &= n >= 4 ? ~0 : (n <= 0 ? 0 : (1 << (8 * n)) - 1);
  }
}

// The same for 16 codes in LDS.
__device__ __forceinline__ void cut16(u32x4* p, int valid) {
  u32x4 w = *p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = valid - 4 * i;
    w[i] &= n >= 4 ? ~0u : (n <= 0 ? 0u : (1u << (8 * n)) - 1);
  }
  *p = w;
}

// What a lane gives to the matrix instructions of a block: its 32 codes, or the same in 16 bits,
// eight for each of four instructions.
template <bool kFull>
struct Operand {
  i32x8 f;
};
template <>
struct Operand<true> {
  bf16x8 f[4];
};

template <bool kFull>
__device__ __forceinline__ Operand<kFull> operand(const i32x8& f) {
  Operand<kFull> o;
  if constexpr (kFull) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)f[i], 1.f, false);
      const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)f[i], 1.f, true);
      const int at = 4 * (i & 1);
      o.f[i / 2][at] = lo[0], o.f[i / 2][at + 1] = lo[1];
      o.f[i / 2][at + 2] = hi[0], o.f[i / 2][at + 3] = hi[1];
    }
  } else {
    o.f = f;
  }
  return o;
}

// Scales as the sums are multiplied by them: an exponent as its power of two.
template <Mode kMode>
__device__ __forceinline__ float factor(uint32_t kept) {
  if constexpr (kMode != kHardware) return __builtin_bit_cast(float, kept);
  return kept == 255 ? NAN : __builtin_bit_cast(float, kept ? kept << 23 : 0x00400000u);
}

// A block's products added to c.
template <Mode kMode, bool kFull>
__device__ __forceinline__ f32x4 block(const Operand<kFull>& b, const Operand<kFull>& a, f32x4 c,
                                       const uint32_t* sb, uint32_t sa) {
  if constexpr (kMode == kHardware && !kFull) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.f, a.f, c, 0, 0, 0, (int)sb[0], 0,
                                                            (int)sa);
  } else {
    f32x4 v = nl2k::zero4();
    if constexpr (kFull) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.f[i], a.f[i], v, 0, 0, 0);
    } else {
      v = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.f, a.f, v, 0, 0, 0, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      c[r] = fmaf(factor<kMode>(sa) * factor<kMode>(sb[kMode == kTiles ? 0 : r]), v[r], c[r]);
    return c;
  }
}

// Scales of b that a lane needs for its sums: its row's, for the instruction; one for all four; or
// four.
template <Mode kMode, bool kFull>
constexpr int scales_of_b() {
  return kMode == kTiles || (kMode == kHardware && !kFull) ? 1 : 4;
}

// `count` of eight numbers of a row of the result.
__device__ __forceinline__ void put8(const Args& g, int64_t at, int count, const float (&v)[8]) {
  if (count <= 0) return;
  if (g.out_dtype == kF32)
    store8<float>(static_cast<float*>(g.out) + at, count, v);
  else if (g.out_dtype == kBF16)
    store8<bf16_t>(static_cast<unsigned short*>(g.out) + at, count, v);
  else
    store8<f16_t>(static_cast<unsigned short*>(g.out) + at, count, v);
}

// BM rows of a by BN of b, WM x WN waves, two stages of 128 bytes a row in LDS.
template <int BM, int BN, int WM, int WN, Mode kMode, bool kFull>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(Args g) {
  constexpr int kWaves = WM * WN;
  constexpr int kRowsAll = BM + BN;
  constexpr int kCodes = kRowsAll * 128;
  constexpr int kStage = kCodes + kRowsAll * 4;       // codes, then a scale for every row
  constexpr int kLoads = kRowsAll / 8 / kWaves;       // of eight rows, a wave and stage
  constexpr int kScaleLoads = kRowsAll / 64 / kWaves;  // of 64 rows' scales
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static_assert(kLoads * 8 * kWaves == kRowsAll && BM % (8 * kWaves) == 0 &&
                    kScaleLoads * 64 * kWaves == kRowsAll && NT % 4 == 0 && BM % 64 == 0,
                "tile shape");
  constexpr int kBytes = kMode == kHardware ? 1 : 4;  // of a scale
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
  const int lane = threadIdx.x & 63, group = lane >> 4, piece = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Workgroups go round the eight XCDs in turn; each XCD is given tiles that lie next to each
  // other, so that its L2 holds the rows they share.
  int x = blockIdx.x;
  {
    const int per = g.tiles >> 3, more = g.tiles & 7, xcd = x & 7;
    x = xcd * per + min(xcd, more) + (x >> 3);
  }
  const int one = g.tiles_a * g.tiles_b;
  const int part = x / one;
  x -= part * one;
  // down four tiles, then across
  const int band = x / (4 * g.tiles_b), top = band * 4, high = min(4, g.tiles_a - top);
  x -= top * g.tiles_b;
  const int tn = x / high, tm = top + x - tn * high;
  const int m0 = tm * BM, n0 = tn * BN;
  const int from = part * g.per, steps = min(g.per, g.steps - from);
  const int left = g.K - (from + steps - 1) * 128;  // numbers of the last step

  // A wave's load fills eight rows of a stage.  The 16-byte pieces of a row are permuted by its
  // number so that the eight rows of which lanes next to each other read a piece lie in
  // different banks: rows 0 .. 7 of a; of b, whose rows a product takes as row_of_b says, four
  // and the four that are 16 on.
  auto key = [](bool second, int row) { return second ? (row & 3) | ((row >> 2) & 4) : row & 7; };
  const uint8_t* abase = scalar_base(g.a.codes + (int64_t)m0 * g.a.pitch + (int64_t)from * 128);
  const uint8_t* bbase = scalar_base(g.b.codes + (int64_t)n0 * g.b.pitch + (int64_t)from * 128);
  uint32_t off[kLoads];
  auto row_of_load = [&](int q) { return (q * kWaves + wave) * 8 + lane / 8; };
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const bool second = q * kWaves * 8 >= BM;
    const int r = row_of_load(q) - (second ? BM : 0);
    const Side& s = second ? g.b : g.a;
    const int last = s.rows - (second ? n0 : m0) - 1;
    off[q] = (uint32_t)min(r, last) * (uint32_t)s.pitch + ((lane & 7) ^ key(second, r)) * 16;
  }
  // rows' scales, 64 a load
  const uint8_t* sbase[kScaleLoads];
  uint32_t soff[kScaleLoads];
#pragma unroll
  for (int q = 0; q < kScaleLoads; ++q) {
    const bool second = (q * kWaves + wave) * 64 >= BM;
    const Side& s = second ? g.b : g.a;
    const int first = second ? n0 : m0;
    const int r = min((q * kWaves + wave) * 64 - (second ? BM : 0) + lane, s.rows - first - 1);
    sbase[q] = scalar_base(s.scales + (int64_t)(first >> s.shift) * s.s_row + from * s.s_block);
    soff[q] = (uint32_t)(((first + r) >> s.shift) - (first >> s.shift)) * (uint32_t)s.s_row;
  }
  const int64_t a_step = g.a.s_block, b_step = g.b.s_block;
  const uint32_t lds0 = offset_of(lds);
  auto load = [&](int s) {
    const uint32_t to = lds0 + (s & 1) * kStage;
    const bool tail = s == steps - 1 && left < 128;
    const int end = ((left + 15) & ~15) - 16;  // the last piece that may be read
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const bool second = q * kWaves * 8 >= BM;
      uint32_t o = off[q];
      if (tail) {
        const int p = ((lane & 7) ^ key(second, row_of_load(q) - (second ? BM : 0))) * 16;
        o -= max(p - end, 0);
      }
      load_lds16(second ? bbase : abase, o,
                 __builtin_amdgcn_readfirstlane(to + (q * kWaves + wave) * 1024));
    }
#pragma unroll
    for (int q = 0; q < kScaleLoads; ++q) {
      load_lds4<kBytes>(sbase[q], soff[q],
                        __builtin_amdgcn_readfirstlane(to + kCodes + (q * kWaves + wave) * 256));
      sbase[q] += (q * kWaves + wave) * 64 >= BM ? b_step : a_step;
    }
    abase += 128;
    bbase += 128;
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = nl2k::zero4();

  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  // Row of b that lane i of 16 holds for product n: four products' sums are then of 16 rows next
  // to each other.  The key of a row does not depend on n, nor that of a's on m.
  auto row_of_b = [&](int n, int i) {
    return wj + (n >> 2) * 64 + 16 * (i >> 2) + 4 * (n & 3) + (i & 3);
  };
  const int ka = key(false, piece), kb = key(true, row_of_b(0, piece));
  const uint8_t* const fa0 = lds + (wi + piece) * 128;
  const uint8_t* const fb0 = lds + (BM + row_of_b(0, piece)) * 128;
  auto read = [&](const uint8_t* row, int k) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(row + ((2 * group) ^ k) * 16);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(row + ((2 * group + 1) ^ k) * 16);
    i32x8 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (int)lo[i], f[4 + i] = (int)hi[i];
    return f;
  };
  constexpr int kB = scales_of_b<kMode, kFull>();

  load(0);
  for (int s = 0; s < steps; ++s) {
    // this wave's share of the stage is there, and its reads of the one before are done; after
    // the barrier all waves'
    wait_reads();
    wait_tile<0>();
    workgroup_barrier();
    if (s + 1 < steps) load(s + 1);
    const int stage = (s & 1) * kStage;
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(lds + stage + kCodes);
    if (s == steps - 1 && left < 128) {  // what lies past the end of a row: zeros
      for (int i = threadIdx.x; i < kRowsAll * 8; i += 64 * kWaves) {
        const int row = i >> 3, r = row < BM ? row : row - BM;
        const int valid = left - ((i & 7) ^ key(row >= BM, r)) * 16;
        if (valid < 16) cut16(reinterpret_cast<u32x4*>(lds + stage + i * 16), valid);
      }
      __syncthreads();
    }
    Operand<kFull> fb[NT];
    uint32_t sb[NT][kB];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      fb[n] = operand<kFull>(read(fb0 + stage + ((n >> 2) * 64 + 4 * (n & 3)) * 128, kb));
      if constexpr (kMode == kTiles) {
        sb[n][0] = scales[BM + wj + (n >> 2) * 64];
      } else if constexpr (kB == 1) {
        sb[n][0] = scales[BM + row_of_b(n, piece)];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) sb[n][r] = scales[BM + row_of_b(n, 4 * group) + r];
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const Operand<kFull> fa = operand<kFull>(read(fa0 + stage + m * 2048, ka));
      const uint32_t sa = scales[wi + m * 16 + piece];
#pragma unroll
      for (int n = 0; n < NT; ++n)
        acc[m][n] = block<kMode, kFull>(fb[n], fa, acc[m][n], sb[n], sa);
    }
  }

  // a lane's 16 sums of a row, next to each other
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = m0 + wi + m * 16 + piece;
    if (row >= g.a.rows) continue;
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      const int col = n0 + row_of_b(n, 4 * group);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[m][n + e / 4][e & 3];
      const int count = g.b.rows - col;
      if (g.partial) {
        if (count > 0)
          store8<float>(g.partial + ((int64_t)part * g.a.rows + row) * g.b.rows + col, count, v);
      } else {
        put8(g, row * g.b.rows + col, count, v);
      }
    }
  }
}

// Few rows of a: 16 rows of b a workgroup, straight to registers, its eight waves taking blocks
// of k in turn and their sums added at the end in a fixed order.  Bound by the reading of b.
constexpr int kThinWaves = 8;

template <int MT, Mode kMode, bool kFull>
__global__ __launch_bounds__(64 * kThinWaves) void thin_kernel(Args g) {
  constexpr int U = MT <= 2 ? 4 : 2;  // blocks in flight
  __shared__ __attribute__((aligned(16))) float sums[kThinWaves][MT * 256];
  const int lane = threadIdx.x & 63, group = lane >> 4, piece = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, part = blockIdx.y;
  const int from = part * g.per, upto = min(from + g.per, g.steps);
  const int left = g.K - (g.steps - 1) * 128;  // numbers of the last block
  const uint32_t end = (uint32_t)((g.K + 15) & ~15) - 16;
  const uint8_t* pb = g.b.codes + (int64_t)min(n0 + piece, g.b.rows - 1) * g.b.pitch;
  const uint8_t* pa[MT];
  const uint8_t* qa[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(m * 16 + piece, g.a.rows - 1);
    pa[m] = g.a.codes + (int64_t)row * g.a.pitch;
    qa[m] = g.a.scales + (int64_t)(row >> g.a.shift) * g.a.s_row;
  }
  constexpr int kB = scales_of_b<kMode, kFull>();
  const uint8_t* qb[kB];
#pragma unroll
  for (int r = 0; r < kB; ++r) {
    // by the instruction: of this lane's row; afterwards: of the rows of its sums
    const int row = kB == 4 ? n0 + 4 * group + r : (kMode == kTiles ? n0 : n0 + piece);
    qb[r] = g.b.scales + (int64_t)(min(row, g.b.rows - 1) >> g.b.shift) * g.b.s_row;
  }
  auto fragment = [&](const uint8_t* p, int s) {
    const uint32_t k = s * 128 + group * 32;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(p + min(k, end));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(p + min(k + 16, end));
    i32x8 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (int)lo[i], f[4 + i] = (int)hi[i];
    return f;
  };
  auto scale = [&](const uint8_t* p, int64_t step, int s) {
    p += s * step;
    return kMode == kHardware ? (uint32_t)*p : *reinterpret_cast<const uint32_t*>(p);
  };
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = nl2k::zero4();
  for (int s0 = from + wave; s0 < upto; s0 += kThinWaves * U) {
    i32x8 fb[U], fa[U][MT];
    uint32_t sb[U][kB], sa[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * kThinWaves, upto - 1);
      fb[u] = fragment(pb, s);
#pragma unroll
      for (int r = 0; r < kB; ++r) sb[u][r] = scale(qb[r], g.b.s_block, s);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        fa[u][m] = fragment(pa[m], s);
        sa[u][m] = scale(qa[m], g.a.s_block, s);
      }
    }
    // All that depends on where k ends comes before the products, and a block past the end is
    // taken as zeros: no branch lies between a product and what reads it.  (Across one, hipcc of
    // ROCm 7.2 left a sum's first reader two instructions behind the matrix instruction, which
    // needs eight: sums were read before they were there.)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * kThinWaves;
      const int valid = s >= upto ? 0 : (s == g.steps - 1 ? left : 128);
      if (valid < 128) {
        cut(fb[u], valid, group);
#pragma unroll
        for (int m = 0; m < MT; ++m) cut(fa[u][m], valid, group);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Operand<kFull> ob = operand<kFull>(fb[u]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[m] =
            block<kMode, kFull>(ob, operand<kFull>(fa[u][m]), acc[m], sb[u], sa[u][m]);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
    *reinterpret_cast<f32x4*>(&sums[wave][m * 256 + piece * 16 + group * 4]) = acc[m];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += 64 * kThinWaves) {
    float v = sums[0][i];
#pragma unroll
    for (int w = 1; w < kThinWaves; ++w) v += sums[w][i];
    const int m = i >> 4, n = n0 + (i & 15);
    if (m >= g.a.rows || n >= g.b.rows) continue;
    const int64_t at = (int64_t)m * g.b.rows + n;
    if (g.partial)
      g.partial[(int64_t)part * g.a.rows * g.b.rows + at] = v;
    else if (g.out_dtype == kF32)
      static_cast<float*>(g.out)[at] = v;
    else
      static_cast<unsigned short*>(g.out)[at] =
          g.out_dtype == kBF16 ? narrow<bf16_t>(v) : narrow<f16_t>(v);
  }
}

// The sums of the parts of k, added in their order.
__global__ __launch_bounds__(256) void join_kernel(Args g, int parts) {
  const int64_t total = (int64_t)g.a.rows * g.b.rows;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= total) return;
  const int count = (int)min((int64_t)8, total - at);
  float v[8];
  values<float>(load8<float>(g.partial + at, count), v);
  for (int p = 1; p < parts; ++p) {
    float w[8];
    values<float>(load8<float>(g.partial + p * total + at, count), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  put8(g, at, count, v);
}

// The kernel and the parts of k for a product's sizes.
struct Plan {
  int tile;   // rows of a and of b a workgroup takes, 0: few rows
  int parts, per;
  int64_t blocks;
};

Plan plan(int64_t M, int64_t N, int64_t K, bool full) {
  const int64_t steps = nl2k::ceil_div(K, 128);
  Plan p{};
  int64_t wanted;
  if (M <= 64) {
    p.tile = 0;
    p.blocks = nl2k::ceil_div(N, 16);
    wanted = std::min(256 / p.blocks, steps / (4 * kThinWaves));
  } else {
    p.tile = !full && nl2k::ceil_div(M, 256) * nl2k::ceil_div(N, 256) >= 192 ? 256 : 128;
    p.blocks = nl2k::ceil_div(M, p.tile) * nl2k::ceil_div(N, p.tile);
    wanted = std::min(256 / p.blocks, steps / 8);
  }
  wanted = std::max(std::min(wanted, (int64_t)16), (int64_t)1);
  p.per = (int)nl2k::ceil_div(steps, wanted);
  p.parts = (int)nl2k::ceil_div(steps, p.per);
  return p;
}

template <Mode kMode, bool kFull>
int launch(const Args& g, const Plan& p, hipStream_t s) {
  if (p.tile == 0) {
    const dim3 grid((uint32_t)p.blocks, (uint32_t)p.parts);
    const int threads = 64 * kThinWaves;
    switch ((g.a.rows + 15) / 16) {
      case 1: thin_kernel<1, kMode, kFull><<<grid, threads, 0, s>>>(g); break;
      case 2: thin_kernel<2, kMode, kFull><<<grid, threads, 0, s>>>(g); break;
      case 3: thin_kernel<3, kMode, kFull><<<grid, threads, 0, s>>>(g); break;
      default: thin_kernel<4, kMode, kFull><<<grid, threads, 0, s>>>(g); break;
    }
  } else if (p.tile == 256) {
    if constexpr (!kFull)
      tile_kernel<256, 256, 2, 4, kMode, kFull><<<dim3((uint32_t)g.tiles), 512, 0, s>>>(g);
  } else {
    tile_kernel<128, 128, 2, 2, kMode, kFull><<<dim3((uint32_t)g.tiles), 256, 0, s>>>(g);
  }
  int st = nl2k::check_launch("block_matmul");
  if (st || p.parts == 1) return st;
  const int64_t n = nl2k::ceil_div((int64_t)g.a.rows * g.b.rows, 8 * 256);
  join_kernel<<<dim3((uint32_t)n), 256, 0, s>>>(g, p.parts);
  return nl2k::check_launch("block_matmul");
}

constexpr int64_t kLongest = 1 << 22;   // numbers of a row: offsets within a tile are of 32 bits

int check_sizes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 1)
    return nl2k::fail(NL2K_ERR_SHAPE, "block_matmul: need M, N >= 0 and K >= 1 (got %lld, %lld, %lld)",
                      (long long)M, (long long)N, (long long)K);
  // tiles of a launch of 512 threads, parts and all
  const int64_t most = nl2k::max_blocks(512) / 16;
  if (M > INT32_MAX - 512 || N > INT32_MAX - 512 || K > kLongest ||
      nl2k::ceil_div(M, 128) * nl2k::ceil_div(N, 128) > most ||
      (M <= 64 && nl2k::ceil_div(N, 16) > most))
    return nl2k::fail(NL2K_ERR_OVERFLOW, "block_matmul: sizes too large (M=%lld N=%lld K=%lld)",
                      (long long)M, (long long)N, (long long)K);
  return NL2K_SUCCESS;
}

size_t workspace_of(const Plan& p, int64_t M, int64_t N) {
  return p.parts > 1 ? (size_t)p.parts * M * N * 4 : 0;
}

int check_side(const char* name, const void* codes, int64_t pitch, const void* scales,
               int64_t row_stride, int64_t block_stride, int scale_type, int64_t rows, int64_t K) {
  if (!codes || !scales)
    return nl2k::fail(NL2K_ERR_NULL, "block_matmul: codes and scales of %s are required", name);
  if (!nl2k::aligned16(codes) ||
      reinterpret_cast<uintptr_t>(scales) % scale_bytes(scale_type))
    return nl2k::fail(NL2K_ERR_ALIGN,
                      "block_matmul: codes of %s must be aligned to 16 bytes, scales to their type",
                      name);
  if (pitch < K || pitch % 16 || pitch > 2 * kLongest)
    return nl2k::fail(NL2K_ERR_SHAPE,
                      "block_matmul: the pitch of %s must be a multiple of 16, at least K and at "
                      "most %lld (got %lld)", name, (long long)(2 * kLongest), (long long)pitch);
  if (row_stride < 0 || block_stride < 0 || row_stride > kLongest ||
      block_stride > INT64_MAX / 16 / kLongest)
    return nl2k::fail(NL2K_ERR_SHAPE, "block_matmul: strides of the scales of %s out of range (%lld, "
                      "%lld)", name, (long long)row_stride, (long long)block_stride);
  (void)rows;
  return NL2K_SUCCESS;
}

}  // namespace

extern "C" size_t block_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int out_dtype) {
  if (check_sizes(M, N, K) || M == 0 || N == 0) return 0;
  return workspace_of(plan(M, N, K, out_dtype == kF32), M, N);
}

extern "C" int block_matmul(const void* a, int64_t a_pitch, const void* a_scales,
                            int64_t a_row_stride, int64_t a_block_stride, int a_tiles,
                            const void* b, int64_t b_pitch, const void* b_scales,
                            int64_t b_row_stride, int64_t b_block_stride, int b_tiles,
                            int scale_type, void* out, int out_dtype, int64_t M, int64_t N,
                            int64_t K, void* workspace, size_t workspace_bytes,
                            hipStream_t stream) {
  int st = check_sizes(M, N, K);
  if (st) return st;
  if (scale_type != kScaleF32 && scale_type != kScaleE8M0)
    return nl2k::fail(NL2K_ERR_VALUE, "block_matmul: scale_type must be 0 or 1 (got %d)",
                      scale_type);
  if (out_dtype < kF32 || out_dtype > kF16)
    return nl2k::fail(NL2K_ERR_VALUE, "block_matmul: out_dtype must be 0, 1 or 2 (got %d)",
                      out_dtype);
  if (M == 0 || N == 0) return nl2k::succeed();
  if ((st = check_side("a", a, a_pitch, a_scales, a_row_stride, a_block_stride, scale_type, M, K)))
    return st;
  if ((st = check_side("b", b, b_pitch, b_scales, b_row_stride, b_block_stride, scale_type, N, K)))
    return st;
  if (!out) return nl2k::fail(NL2K_ERR_NULL, "block_matmul: out is required");
  if (reinterpret_cast<uintptr_t>(out) % bytes_of(out_dtype))
    return nl2k::fail(NL2K_ERR_ALIGN, "block_matmul: out must be aligned to its type");
  const Plan p = plan(M, N, K, out_dtype == kF32);
  const size_t need = workspace_of(p, M, N);
  if (need && (!workspace || workspace_bytes < need))
    return nl2k::fail(NL2K_ERR_WORKSPACE, "block_matmul: needs a workspace of %zu bytes (got %zu)",
                      need, workspace_bytes);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 4)
    return nl2k::fail(NL2K_ERR_ALIGN, "block_matmul: the workspace must be aligned to 4 bytes");
  const int64_t e = scale_bytes(scale_type);
  auto side = [&](const void* c, int64_t pitch, const void* s, int64_t row, int64_t block,
                  int tiles, int64_t rows) {
    return Side{static_cast<const uint8_t*>(c), static_cast<const uint8_t*>(s), pitch, row * e,
                block * e, (int32_t)rows, tiles ? 7 : 0};
  };
  Args g{};
  g.a = side(a, a_pitch, a_scales, a_row_stride, a_block_stride, a_tiles, M);
  g.b = side(b, b_pitch, b_scales, b_row_stride, b_block_stride, b_tiles, N);
  g.out = out;
  g.partial = need ? static_cast<float*>(workspace) : nullptr;
  g.K = (int32_t)K;
  g.steps = (int32_t)nl2k::ceil_div(K, 128);
  g.per = p.per;
  g.out_dtype = out_dtype;
  if (p.tile) {
    g.tiles_a = (int32_t)nl2k::ceil_div(M, p.tile);
    g.tiles_b = (int32_t)nl2k::ceil_div(N, p.tile);
    g.tiles = (int32_t)(p.blocks * p.parts);
  }
  const bool full = out_dtype == kF32;
  if (scale_type == kScaleE8M0)
    return full ? launch<kHardware, true>(g, p, stream) : launch<kHardware, false>(g, p, stream);
  if (b_tiles)
    return full ? launch<kTiles, true>(g, p, stream) : launch<kTiles, false>(g, p, stream);
  return full ? launch<kRows, true>(g, p, stream) : launch<kRows, false>(g, p, stream);
}

extern "C" const char* block_matmul_last_error(void) { return nl2k::error_slot().text; }
