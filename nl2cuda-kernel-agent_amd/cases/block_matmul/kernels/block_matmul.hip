// Products of e4m3 matrices with a scale for each block of 128, for MI355X
// (gfx950).  C-ABI in include/block_matmul.h.
//
// The matrix instruction takes 16 rows of each operand and 128 numbers of k, a
// block: 32 a lane, lane l of row l % 16; which 32 does not matter, so long as both
// operands' lanes hold the same: the 16 from 16 (l / 16) on and those from 64 on
// after them, so that four lanes read 64 bytes of a row.  b's rows are its
// first operand and a's its second, so that a lane's sums are of one row of a
// and of numbers next to each other in a row of the result.
//
// Scales that are powers of two the instruction applies itself.  32-bit ones
// are applied to a block's sums, in registers: sum += (sa sb) block.
//
// The 8-bit instruction adds eight products at a time in a narrow window: what
// lies 13 bits below the largest of the eight is dropped.  A result is off by at
// most 7 2^-13 of the sum of the eights' largest products, also where it is small
// itself; of random numbers by 1.5e-5 of the results' root mean square (measured;
// 9.8e-9 with the 16-bit instruction).  Rounding costs 1.7e-3 of it in bfloat16 and
// 2.1e-4 in float16, so 16-bit results are computed with it.  For 32-bit results
// the codes become bfloat16, which holds them exactly, and the 16-bit
// instruction, at half the rate, keeps every product whole; with the conversions
// it takes 2.5 times as long.

#include "block_matmul.h"

#include "e4m3.h"
#include "lds_direct.h"
#include "quantize.h"

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
  int32_t K, steps;  // numbers of a row, and its blocks
  int32_t per;     // blocks of k of a part
  int32_t tiles_a, tiles_b, tiles;
  int out_dtype;
};

// Lane group g's 32 numbers of a block of which `valid` count: the others 0.
__device__ __forceinline__ void cut(i32x8& f, int valid, int group) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = valid - (i < 4 ? 0 : 64) - 16 * group - 4 * (i & 3);
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

// Whether scales are applied to a block's sums, and how many of b's a lane then needs for its four:
// one, or four; the instruction takes that of the lane's row.
template <Mode kMode, bool kFull>
constexpr bool applied_later() {
  return kMode != kHardware || kFull;
}
template <Mode kMode, bool kFull>
constexpr int scales_of_b() {
  return kMode == kTiles || !applied_later<kMode, kFull>() ? 1 : 4;
}

__device__ __forceinline__ float as_float(uint32_t bits) {
  return __builtin_bit_cast(float, bits);
}

// A scale as it is read, for the instruction or as the bits of what sums are multiplied by.
template <Mode kMode, bool kFull>
__device__ __forceinline__ uint32_t ready(uint32_t kept) {
  if constexpr (kMode != kHardware || !kFull) return kept;
  // 2^-127 is half of what `kept` << 23 begins with, and infinity times 0 makes 255 a NaN
  const float f = as_float(max(kept << 23, 0x00400000u));
  return __builtin_bit_cast(uint32_t, fmaf(f, 0.f, f));
}

// A block's products, without scales.
template <bool kFull>
__device__ __forceinline__ f32x4 sums(const Operand<kFull>& b, const Operand<kFull>& a) {
  f32x4 v = nl2k::zero4();
  if constexpr (kFull) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.f[i], a.f[i], v, 0, 0, 0);
  } else {
    v = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.f, a.f, v, 0, 0, 0, 0, 0, 0);
  }
  return v;
}

// A block's products, scaled and added to c.
template <Mode kMode, bool kFull>
__device__ __forceinline__ f32x4 block(const Operand<kFull>& b, const Operand<kFull>& a, f32x4 c,
                                       const uint32_t* sb, uint32_t sa) {
  if constexpr (!applied_later<kMode, kFull>()) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.f, a.f, c, 0, 0, 0, (int)sb[0], 0,
                                                            (int)sa);
  } else {
    const f32x4 v = sums<kFull>(b, a);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      c[r] = fmaf(as_float(sa) * as_float(sb[kMode == kTiles ? 0 : r]), v[r], c[r]);
    return c;
  }
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

// One sum.
__device__ __forceinline__ void put1(const Args& g, int part, int64_t row, int64_t col, float v) {
  const int64_t at = row * g.b.rows + col;
  if (g.partial)
    g.partial[(int64_t)part * g.a.rows * g.b.rows + at] = v;
  else if (g.out_dtype == kF32)
    static_cast<float*>(g.out)[at] = v;
  else
    static_cast<unsigned short*>(g.out)[at] =
        g.out_dtype == kBF16 ? narrow<bf16_t>(v) : narrow<f16_t>(v);
}

// The pieces of 16 bytes of a row in LDS are permuted by the row's number, so that the 64 banks
// give a wave its 1024 bytes in four clocks: lanes read pieces `group` and `group` + 4 of 16 rows
// (pieces 2 group and 2 group + 1 took eight).
__device__ __forceinline__ i32x8 read_row(const uint8_t* row, int group, int key) {
  const u32x4 lo = *reinterpret_cast<const u32x4*>(row + (group ^ key) * 16);
  const u32x4 hi = *reinterpret_cast<const u32x4*>(row + ((group + 4) ^ key) * 16);
  i32x8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = (int)lo[i], f[4 + i] = (int)hi[i];
  return f;
}

// All of this wave's reads of LDS are done and all but N of its loads have arrived; after the
// barrier all waves'.
template <int N>
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_sched_barrier(0);
  wait_reads();
  wait_tile<N>();
  workgroup_barrier();
}

// BM x BN tiles of WM x WN waves, S stages of 128 bytes a row in LDS.
//
// A wave goes through its rows of a with all its rows of b in registers.  The last kLast rows of a
// it keeps back: once every wave has read the stage for the last time, these are multiplied column
// by column, and between them the next stage's rows of b come into the registers that become free.
// So the barrier, and the reads after it, lie under products; a stage's loads have S - 1 stages'
// time.  The loop has no branch, since with one the compiler no longer keeps everything in registers:
// the last block of k, inside which rows may end, is taken first and its zeros are put in before the
// loop, and past the last stage the last one is loaded again, to where nobody reads.
//
// Bound by power: 8192 x 8192 x 8192 takes 410 us, 2680 TFLOP/s, at a clock that falls to 1.8 GHz,
// the matrix cores busy 68 in 100 clocks; with 32-bit scales for tiles 447 us, for rows 510.  Scales
// that are applied afterwards are two products behind, which hides them: 495 and 575 us at once
// after each product; for tiles one scale is read and one factor formed for four products, 453 us for
// 461 then.  Four waves of 128 x 128 took 445 us, b straight to registers 764.
// 128 x 128 tiles, for smaller products, wait for LDS: eight waves and four stages take 19 us for
// 512 x 4096 x 4096 and 35 for 3000 x 1000 x 8192, with two stages 24 and 44, four waves with two or
// four stages 26 and 47.  256 x 128 with three stages 36 us for 2048 x 4096 x 4096, with two 37.
// Precise products are bound by vector instructions, 128 conversions, 64 additions and 4 or 64
// multiplications of scales for 64 matrix instructions: 8192 x 8192 x 8192 1015 us, with 32-bit
// scales for tiles 937.  The second number of __launch_bounds__ leaves a wave no registers but those
// that vector instructions read, without which each sum is moved there: 1072 us for 1144, and 962
// for 1029.
template <int BM, int BN, int WM, int WN, int kLast, int S, Mode kMode, bool kFull>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(Args g) {
  constexpr int kWaves = WM * WN;
  constexpr int kRowsAll = BM + BN;
  constexpr int kCodes = kRowsAll * 128;
  constexpr int kStage = kCodes + kRowsAll * 4;  // codes, then a scale for every row
  constexpr int kLoads = kRowsAll / 8 / kWaves;  // of eight rows, a wave and stage
  constexpr int kScaleParts = kRowsAll / 64;     // loads of 64 rows' scales
  constexpr int kScaleLoads = (kScaleParts + kWaves - 1) / kWaves;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static_assert(kLoads * 8 * kWaves == kRowsAll && BM % (8 * kWaves) == 0 && NT % 4 == 0 &&
                    BM % 64 == 0 && BN % 64 == 0 && kLast > 1 && kLast <= MT,
                "tile shape");
  constexpr int kBytes = kMode == kHardware ? 1 : 4;  // of a scale
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S * kStage];
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
  const int64_t last_block = from + steps - 1;
  const int left = min(g.K - (int)last_block * 128, 128);  // numbers of it

  // A wave's load fills eight rows.  Keys of rows: of a, its number; of b, whose rows a product
  // takes as row_of_b says, four rows and the four that are 16 on.
  auto key = [](bool second, int row) { return second ? (row & 3) | ((row >> 2) & 4) : row & 7; };
  const uint8_t* abase = scalar_base(g.a.codes + (int64_t)m0 * g.a.pitch + last_block * 128);
  const uint8_t* bbase = scalar_base(g.b.codes + (int64_t)n0 * g.b.pitch + last_block * 128);
  auto row_of_load = [&](int q) {
    return (q * kWaves + wave) * 8 + lane / 8 - (q * kWaves * 8 >= BM ? BM : 0);
  };
  auto piece_of_load = [&](int q) {
    return ((lane & 7) ^ key(q * kWaves * 8 >= BM, row_of_load(q))) * 16;
  };
  // by how much a lane's piece lies past the last that may be read of the last block
  auto past_end = [&](int q) {
    return (uint32_t)max(piece_of_load(q) - (((left + 15) & ~15) - 16), 0);
  };
  uint32_t off[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const bool second = q * kWaves * 8 >= BM;
    const Side& s = second ? g.b : g.a;
    // rows past the operand's last are copies of it, whose sums are not stored
    const int row = min(row_of_load(q), s.rows - (second ? n0 : m0) - 1);
    off[q] = (uint32_t)row * (uint32_t)s.pitch + piece_of_load(q) - past_end(q);
  }
  const uint8_t* sbase[kScaleLoads];
  uint32_t soff[kScaleLoads];
  auto scale_part = [&](int q) { return min(q * kWaves + wave, kScaleParts - 1); };
#pragma unroll
  for (int q = 0; q < kScaleLoads; ++q) {
    const bool second = scale_part(q) * 64 >= BM;
    const Side& s = second ? g.b : g.a;
    const int first = second ? n0 : m0;
    const int r = min(scale_part(q) * 64 - (second ? BM : 0) + lane, s.rows - first - 1);
    sbase[q] = scalar_base(s.scales + (int64_t)(first >> s.shift) * s.s_row +
                           last_block * s.s_block);
    soff[q] = (uint32_t)(((first + r) >> s.shift) - (first >> s.shift)) * (uint32_t)s.s_row;
  }
  const int64_t a_step = g.a.s_block, b_step = g.b.s_block;
  const uint32_t lds0 = offset_of(lds);
  auto load_some = [&](uint32_t stage, int q0, int q1) {
    const uint32_t to = lds0 + stage;
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      if (q >= q0 && q < q1)
        load_lds16(q * kWaves * 8 >= BM ? bbase : abase, off[q],
                   __builtin_amdgcn_readfirstlane(to + (q * kWaves + wave) * 1024));
  };
  // the scales, and on to the next block: after the last the first
  auto load_rest = [&](uint32_t stage, int s) {
    const uint32_t to = lds0 + stage;
    const int64_t by = s == 0 ? 1 - steps : s + 1 < steps ? 1 : 0;
#pragma unroll
    for (int q = 0; q < kScaleLoads; ++q) {
      load_lds4<kBytes>(sbase[q], soff[q],
                        __builtin_amdgcn_readfirstlane(to + kCodes + scale_part(q) * 256));
      sbase[q] += by * (scale_part(q) * 64 >= BM ? b_step : a_step);
    }
    abase += by * 128;
    bbase += by * 128;
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
  constexpr int kB = scales_of_b<kMode, kFull>();
  Operand<kFull> fb[NT], fa[kLast];  // row m of a in fa[m % kLast]
  uint32_t sb[NT][kB], sa[kLast];
  auto get_b = [&](int stage, int n) {
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(lds + stage + kCodes) + BM;
    fb[n] = operand<kFull>(
        read_row(fb0 + stage + ((n >> 2) * 64 + 4 * (n & 3)) * 128, group, kb));
    if constexpr (kMode == kTiles) {  // four products' rows lie in one tile
      if (n % 4 == 0) sb[n][0] = scales[wj + n * 16];
    } else {
#pragma unroll
      for (int r = 0; r < kB; ++r)
        sb[n][r] = ready<kMode, kFull>(
            scales[kB == 1 ? row_of_b(n, piece) : row_of_b(n, 4 * group) + r]);
    }
  };
  auto get_a = [&](int stage, int m) {
    fa[m % kLast] = operand<kFull>(read_row(fa0 + stage + m * 2048, group, ka));
    sa[m % kLast] = ready<kMode, kFull>(
        reinterpret_cast<const uint32_t*>(lds + stage + kCodes)[wi + m * 16 + piece]);
  };

  // Product j of a stage: rows one after the other, the last ones column by column.
  constexpr int kFirst = (MT - kLast) * NT;
  auto row_of = [&](int j) { return j < kFirst ? j / NT : MT - kLast + (j - kFirst) % kLast; };
  auto col_of = [&](int j) { return j < kFirst ? j % NT : (j - kFirst) / kLast; };
  // Scales that are applied afterwards: two products behind, while the next ones run.
  constexpr bool kLater = applied_later<kMode, kFull>();
  constexpr int kBehind = 2;
  f32x4 ring[kBehind];
  float factors[kMode == kTiles ? MT * NT / 4 : kBehind][kB];
  auto factor_of = [&](int j) {
    return kMode == kTiles ? row_of(j) * (NT / 4) + col_of(j) / 4 : j % kBehind;
  };
  auto retire = [&](int j) {
    const int m = row_of(j), n = col_of(j);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      acc[m][n][r] =
          fmaf(factors[factor_of(j)][kB == 1 ? 0 : r], ring[j % kBehind][r], acc[m][n][r]);
  };
  auto multiply = [&](int j) {
    const int m = row_of(j), n = col_of(j);
    if constexpr (!kLater) {
      acc[m][n] = block<kMode, kFull>(fb[n], fa[m % kLast], acc[m][n], sb[n], sa[m % kLast]);
    } else {
      if (j >= kBehind) retire(j - kBehind);
      if (kMode != kTiles || n % 4 == 0) {
#pragma unroll
        for (int r = 0; r < kB; ++r)
          factors[factor_of(j)][r] = as_float(sa[m % kLast]) * as_float(sb[n][r]);
      }
      ring[j % kBehind] = sums<kFull>(fb[n], fa[m % kLast]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  load_some(0, 0, kLoads);
  if (steps > 1) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) off[q] += past_end(q);
  }
  load_rest(0, 0);
#pragma unroll
  for (int s = 1; s < S; ++s) {
    load_some(s * kStage, 0, kLoads);
    load_rest(s * kStage, s);
  }
  arrive<(S - 1) * (kLoads + kScaleLoads)>();
  if (left < 128) {  // zeros where rows have ended
    for (int i = threadIdx.x; i < kRowsAll * 8; i += 64 * kWaves) {
      const int row = i >> 3;
      const int valid = left - ((i & 7) ^ key(row >= BM, row < BM ? row : row - BM)) * 16;
      if (valid < 16) cut16(reinterpret_cast<u32x4*>(lds + i * 16), valid);
    }
    wait_reads();
    workgroup_barrier();
  }
  get_a(0, 0);
#pragma unroll
  for (int n = 0; n < NT; ++n) get_b(0, n);
  for (int s = 0; s < steps; ++s) {
    const int at = s % S * kStage, next = (s + 1) % S * kStage;
#pragma unroll
    for (int m = 0; m < MT - kLast; ++m) {
      get_a(at, m + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NT; ++n) multiply(m * NT + n);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = MT - kLast + 1; m < MT; ++m) get_a(at, m);
    arrive<(S - 2) * (kLoads + kScaleLoads)>();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      load_some(at, n * kLoads / NT, (n + 1) * kLoads / NT);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < kLast; ++m) multiply(kFirst + n * kLast + m);
      __builtin_amdgcn_sched_barrier(0);
      get_b(next, n);
      if (n == NT - 1) get_a(next, 0);
    }
    load_rest(at, s + S);
    if constexpr (kLater) {
#pragma unroll
      for (int j = MT * NT - kBehind; j < MT * NT; ++j) retire(j);
    }
  }
  wait_tile<0>();  // nothing is on its way to LDS when it is given back

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

// Few rows of a, many numbers of b: 64 rows of b a workgroup of four waves, S stages of 128 bytes a
// row in LDS, so that 100 KB a CU are on their way.  Bound by the reading of b: 37 rows times 16384 x
// 2048 8.8 us, times 8192 x 4096 11.5, where thin_kernel, which reads a from L2 for every 16 rows of
// b, takes 15.8 and 15.9.
template <int MT, int S, Mode kMode, bool kFull>
__global__ __launch_bounds__(256) void slim_kernel(Args g) {
  constexpr int kWaves = 4, BM = (MT * 16 + 31) / 32 * 32, BN = 64, kRowsAll = BM + BN;
  constexpr int kCodes = kRowsAll * 128, kStage = kCodes + 128 * 4;
  constexpr int kLoads = kRowsAll / 8 / kWaves;
  constexpr int kBytes = kMode == kHardware ? 1 : 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S * kStage];
  const int lane = threadIdx.x & 63, group = lane >> 4, piece = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * BN, part = blockIdx.y;
  const int from = part * g.per, steps = min(g.per, g.steps - from);
  const int64_t last_block = from + steps - 1;  // taken first, as in tile_kernel
  const int left = min(g.K - (int)last_block * 128, 128);
  const uint8_t* abase = scalar_base(g.a.codes + last_block * 128);
  const uint8_t* bbase = scalar_base(g.b.codes + (int64_t)n0 * g.b.pitch + last_block * 128);
  const int swapped = ((lane & 7) ^ (lane >> 3)) * 16;
  const uint32_t past = (uint32_t)max(swapped - (((left + 15) & ~15) - 16), 0);
  uint32_t off[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const bool second = q * kWaves * 8 >= BM;
    const Side& s = second ? g.b : g.a;
    const int r = (q * kWaves + wave) * 8 + lane / 8 - (second ? BM : 0);
    off[q] = (uint32_t)min(r, s.rows - (second ? n0 : 0) - 1) * (uint32_t)s.pitch + swapped - past;
  }
  // scales: a's by the first and the third wave, b's by the others
  const bool sb_wave = wave & 1;
  const Side& ss = sb_wave ? g.b : g.a;
  const int sfirst = sb_wave ? n0 : 0;
  const int sr = min(lane, ss.rows - sfirst - 1);
  const uint8_t* sbase = scalar_base(ss.scales + (int64_t)(sfirst >> ss.shift) * ss.s_row +
                                     last_block * ss.s_block);
  const uint32_t soff =
      (uint32_t)(((sfirst + sr) >> ss.shift) - (sfirst >> ss.shift)) * (uint32_t)ss.s_row;
  const int64_t sstep = ss.s_block;
  const uint32_t lds0 = offset_of(lds);
  uint32_t to = lds0;
  int done = 0;
  auto load = [&]() {
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      load_lds16(q * kWaves * 8 >= BM ? bbase : abase, off[q],
                 __builtin_amdgcn_readfirstlane(to + (q * kWaves + wave) * 1024));
    load_lds4<kBytes>(sbase, soff, __builtin_amdgcn_readfirstlane(to + kCodes + (wave & 1) * 256));
    const int64_t by = done == 0 ? 1 - steps : done + 1 < steps ? 1 : 0;
    ++done;
    abase += by * 128;
    bbase += by * 128;
    sbase += by * sstep;
    to += kStage;
    if (to == lds0 + S * kStage) to = lds0;
  };
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = nl2k::zero4();
  const int ka = piece & 7;
  const uint8_t* const fa0 = lds + piece * 128;
  const uint8_t* const fb0 = lds + (BM + wave * 16 + piece) * 128;
  constexpr int kB = scales_of_b<kMode, kFull>();
  load();
  if (steps > 1) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) off[q] += past;
  }
#pragma unroll
  for (int s = 1; s < S - 1; ++s) load();
  int stage = 0;
  for (int s = 0; s < steps; ++s) {
    arrive<(S - 2) * (kLoads + 1)>();
    load();
    if (s == 0 && left < 128) {
      for (int i = threadIdx.x; i < kRowsAll * 8; i += 64 * kWaves) {
        const int valid = left - ((i & 7) ^ ((i >> 3) & 7)) * 16;
        if (valid < 16) cut16(reinterpret_cast<u32x4*>(lds + i * 16), valid);
      }
      wait_reads();
      workgroup_barrier();
    }
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(lds + stage + kCodes);
    const Operand<kFull> fb = operand<kFull>(read_row(fb0 + stage, group, ka));
    uint32_t sb[kB];
#pragma unroll
    for (int r = 0; r < kB; ++r)
      sb[r] = ready<kMode, kFull>(
          scales[64 + wave * 16 + (kB == 4 ? 4 * group + r : (kMode == kTiles ? 0 : piece))]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      acc[m] = block<kMode, kFull>(
          fb, operand<kFull>(read_row(fa0 + stage + m * 2048, group, ka)), acc[m], sb,
          ready<kMode, kFull>(scales[m * 16 + piece]));
    stage += kStage;
    if (stage == S * kStage) stage = 0;
  }
  wait_tile<0>();
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = m * 16 + piece, col = n0 + wave * 16 + 4 * group;
    if (row >= g.a.rows) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < g.b.rows) put1(g, part, row, col + r, acc[m][r]);
  }
}

// Few rows, or small products: MT times 16 rows of a and NT times 16 of b a workgroup, straight to
// registers, its eight waves taking U blocks of k in turn, the next ones on their way, and their sums
// added at the end in a fixed order.  Few rows are bound by the reading of b: one row times 8192 x
// 4096 7.7 us (4.4 TB/s), times 4096 x 14336 10.8 (5.4).  Small products are bound by the loads'
// latency, eight blocks' at a time where tile_kernel's is each block's, who starts with 4 us of first
// loads and barriers: 384 x 256 x 1423 5.0 us for 10.1.  64 x 64 did not fit in registers, 31 us for
// 225 x 1125 x 3320 where 64 x 32 takes 12.
constexpr int kThinWaves = 8;

template <int MT, int NT, int U, Mode kMode, bool kFull>
__global__ __launch_bounds__(64 * kThinWaves) void thin_kernel(Args g) {
  constexpr int kChunks = NT * 4;  // of four sums, in a row
  __shared__ f32x4 red[kThinWaves][MT * 16 * kChunks];
  const int lane = threadIdx.x & 63, group = lane >> 4, piece = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ta = NT > 1 ? (int)blockIdx.x / g.tiles_b : 0, part = blockIdx.y;
  const int m0 = ta * MT * 16, n0 = ((int)blockIdx.x - ta * g.tiles_b) * NT * 16;
  const int from = part * g.per, upto = min(from + g.per, g.steps);
  const int left = g.K - (g.steps - 1) * 128;  // numbers of the last block
  const uint32_t end = (uint32_t)((g.K + 15) & ~15) - 16;
  constexpr int kB = scales_of_b<kMode, kFull>();
  const uint8_t* abase = scalar_base(g.a.codes + (int64_t)m0 * g.a.pitch);
  const uint8_t* bbase = scalar_base(g.b.codes + (int64_t)n0 * g.b.pitch);
  const uint8_t* sabase = scalar_base(g.a.scales + (int64_t)(m0 >> g.a.shift) * g.a.s_row);
  const uint8_t* sbbase = scalar_base(g.b.scales + (int64_t)(n0 >> g.b.shift) * g.b.s_row);
  // of the rows that a lane reads, and of their scales; rows past the last are copies of it
  uint32_t offa[MT], offb[NT], sca[MT], scb[NT][kB];
  auto scale_at = [](const Side& s, int first, int row) {
    return (uint32_t)((row >> s.shift) - (first >> s.shift)) * (uint32_t)s.s_row;
  };
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = min(m0 + m * 16 + piece, g.a.rows - 1);
    offa[m] = (uint32_t)(row - m0) * (uint32_t)g.a.pitch;
    sca[m] = scale_at(g.a, m0, row);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = min(n0 + n * 16 + piece, g.b.rows - 1);
    offb[n] = (uint32_t)(row - n0) * (uint32_t)g.b.pitch;
#pragma unroll
    for (int r = 0; r < kB; ++r) {
      const int of = n0 + n * 16 + (kB == 4 ? 4 * group + r : (kMode == kTiles ? 0 : piece));
      scb[n][r] = scale_at(g.b, n0, min(of, g.b.rows - 1));
    }
  }
  auto fragment = [&](const uint8_t* base, uint32_t off, int s) {
    const uint32_t k = s * 128 + group * 16;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(base + (off + min(k, end)));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(base + (off + min(k + 64, end)));
    i32x8 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (int)lo[i], f[4 + i] = (int)hi[i];
    return f;
  };
  auto scale = [&](const uint8_t* base, uint32_t off, int64_t step, int s) {
    const uint8_t* p = base + s * step;
    return ready<kMode, kFull>(kMode == kHardware
                                   ? (uint32_t)p[off]
                                   : *reinterpret_cast<const uint32_t*>(p + off));
  };
  struct Batch {
    i32x8 fb[U][NT], fa[U][MT];
    uint32_t sb[U][NT][kB], sa[U][MT];
  };
  auto fetch = [&](int s0, Batch& t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * kThinWaves, upto - 1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        t.fb[u][n] = fragment(bbase, offb[n], s);
#pragma unroll
        for (int r = 0; r < kB; ++r) t.sb[u][n][r] = scale(sbbase, scb[n][r], g.b.s_block, s);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        t.fa[u][m] = fragment(abase, offa[m], s);
        t.sa[u][m] = scale(sabase, sca[m], g.a.s_block, s);
      }
    }
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = nl2k::zero4();
  auto use = [&](int s0, Batch& t) {
    // All that depends on where k ends comes before the products, and a block past the end is
    // taken as zeros, so that the products of all blocks and the scaling of their sums follow each
    // other without a branch: in an earlier form, with one among them, sums were read before they
    // were there.  Where the instruction applies scales, what reads its sums first lies behind the
    // loop's exit; the compiler counts its waits across that branch, and a test reads the built
    // kernels for them.
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * kThinWaves;
      const int valid = s >= upto ? 0 : (s == g.steps - 1 ? left : 128);
      if (valid < 128) {
#pragma unroll
        for (int n = 0; n < NT; ++n) cut(t.fb[u][n], valid, group);
#pragma unroll
        for (int m = 0; m < MT; ++m) cut(t.fa[u][m], valid, group);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Operand<kFull> ob[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) ob[n] = operand<kFull>(t.fb[u][n]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const Operand<kFull> oa = operand<kFull>(t.fa[u][m]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          acc[m][n] = block<kMode, kFull>(ob[n], oa, acc[m][n], t.sb[u][n], t.sa[u][m]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  Batch t0, t1;
  int s0 = from + wave;
  fetch(s0, t0);
  while (s0 < upto) {
    if (s0 + kThinWaves * U < upto) fetch(s0 + kThinWaves * U, t1);
    use(s0, t0);
    s0 += kThinWaves * U;
    if (s0 >= upto) break;
    if (s0 + kThinWaves * U < upto) fetch(s0 + kThinWaves * U, t0);
    use(s0, t1);
    s0 += kThinWaves * U;
  }
  // chunks permuted by their row, so that 16 rows' lie in all banks
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      red[wave][(m * 16 + piece) * kChunks + ((n * 4 + group) ^ (piece & (kChunks - 1)))] =
          acc[m][n];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * kChunks * 4; i += 64 * kThinWaves) {
    const int row = i / (kChunks * 4), col = i - row * (kChunks * 4);
    const int at = row * kChunks + ((col >> 2) ^ (row & (kChunks - 1)));
    float v = red[0][at][col & 3];
#pragma unroll
    for (int w = 1; w < kThinWaves; ++w) v += red[w][at][col & 3];
    const int m = m0 + row, n = n0 + col;
    if (m < g.a.rows && n < g.b.rows) put1(g, part, m, n, v);
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
enum Kernel { kThin, kSmall, kSlim, kTile128, kTile256x128, kTile256 };

constexpr int64_t kMostParts = 16;

struct Plan {
  Kernel kernel;
  int bm, bn;        // rows of a and of b a workgroup takes
  int parts, per;    // parts of k, and the blocks of one
  int64_t blocks;    // workgroups of a part
};

Plan plan(int64_t M, int64_t N, int64_t K, bool full) {
  const int64_t steps = nl2k::ceil_div(K, kBlock);
  auto divide = [&](Kernel kernel, int bm, int bn, int64_t wanted) {
    Plan p{};
    p.kernel = kernel, p.bm = bm, p.bn = bn;
    p.blocks = nl2k::ceil_div(M, bm) * nl2k::ceil_div(N, bn);
    wanted = std::max(std::min(wanted, std::min(steps, kMostParts)), (int64_t)1);
    p.per = (int)nl2k::ceil_div(steps, wanted);
    p.parts = (int)nl2k::ceil_div(steps, p.per);
    return p;
  };
  if (M <= 64) {
    const int64_t n64 = nl2k::ceil_div(N, 64), n16 = nl2k::ceil_div(N, 16);
    // A workgroup for every 16 rows of b has more of them in the air, one for every 64 reads a less
    // often; us, the first against the second: 37 rows times 2048 x 2048 5.5, 7.2, 4096 x 14336 24.7,
    // 15.6; 16 rows times 8192 x 8192 17.3, 14.4, 28672 x 8192 58, 45, 6000 x 6000 11.2, 11.9.  Where
    // the second are one round of the CUs, fewer rows too: 8 times 14336 x 4096 14.5, 10.9, one 12.2,
    // 11.1; but one times 11008 x 4096 (two thirds of a round, 32-bit scales) 10.2, 11.2, times 28672 x
    // 4096 22.1, 24.6.
    const bool one_round = n64 > 200 && n64 <= 256 && N * K >= (int64_t)1 << 25;
    if (one_round || (M > 8 && N * K > (int64_t)(M > 16 ? 2 : 5) << 23))
      return divide(kSlim, 64, 64, 256 / n64);
    // parts of k as CUs are idle, but no shorter than pays for the second launch: 64 rows times 512 x
    // 16384 in 8 parts 12.0, in 4 15.1; 17 times 2048 x 4096 in one part 6.4, in two 7.0
    return divide(kThin, 64, 16, std::min(256 / n16, steps / (M > 32 ? 16 : 30)));
  }
  // Microseconds of a stage on an idle chip, and on one whose every CU has a tile, or two of the
  // precise ones, whose products leave registers for 128 x 128 alone; what a tile begins and ends
  // with; all with scales in 8 bits.  Measured against the others in us, 256 x 256, 256 x 128 and
  // 128 x 128: 4096 x 4096 x 4096 58, 71, 85; 2048 x 4096 x 4096 47, 38, 43; 1024 x 4096 x 4096 45,
  // 29, 23; 256 x 8192 x 8192 with k in two parts 55, 38, 31, whole 80, 48, 32.  64 x 32, whose stage
  // is eight blocks of k, one for each wave, against 128 x 128: 386 x 1128 x 1581 6.0, 10.7, with
  // float32 results 9.1, 17.5; 147 x 3085 x 5632 28, 18.
  struct Tile {
    Kernel kernel;
    int bm, bn, blocks, a_round;
    double idle, busy, once;
  };
  static const Tile kFast[] = {{kTile256, 256, 256, 1, 256, 1.2, 1.7, 7.0},
                               {kTile256x128, 256, 128, 1, 256, 0.72, 1.1, 5.5},
                               {kTile128, 128, 128, 1, 256, 0.47, 0.65, 4.0},
                               {kSmall, 64, 32, 8, 256, 2.4, 2.5, 1.0}};
  static const Tile kPrecise[] = {{kTile128, 128, 128, 1, 512, 1.25, 2.1, 4.0},
                                  {kSmall, 64, 32, 8, 256, 3.2, 3.3, 1.0}};
  Plan best{};
  double least = 1e30;
  for (int i = 0; i < (full ? 2 : 4); ++i) {
    const Tile& t = full ? kPrecise[i] : kFast[i];
    for (int64_t wanted = 1; wanted <= kMostParts; ++wanted) {
      const Plan p = divide(t.kernel, t.bm, t.bn, wanted);
      const int64_t n = p.blocks * p.parts, rounds = nl2k::ceil_div(n, t.a_round);
      const double share = t.a_round == 256 ? std::min(n / 256.0, 1.0) : (n > 256 ? 1.0 : 0.0);
      const double stages = (double)nl2k::ceil_div(p.per, t.blocks);
      double us = (double)rounds * (stages * (t.idle + (t.busy - t.idle) * share * share) + t.once);
      // the parts' sums: a launch, and their bytes
      if (p.parts > 1) us += 3.0 + 2e-6 * (double)p.parts * (double)(M * N);
      if (us < least) least = us, best = p;
    }
  }
  return best;
}

template <Mode kMode, bool kFull>
int launch(const Args& g, const Plan& p, hipStream_t s) {
  const dim3 grid((uint32_t)p.blocks, (uint32_t)p.parts), tiles((uint32_t)g.tiles);
  const int mt = (g.a.rows + 15) / 16;
  if (p.kernel == kThin) {
    const int threads = 64 * kThinWaves;
    // two blocks at a time where a wave has three to eight: 7.6 us for 8.3 at 32 blocks of 8192 rows,
    // but 8.3 for 7.5 at 16 of 16384 rows and 12.9 for 12.2 at 112 of 4096; precise ones would have
    // registers for one workgroup a CU alone, 11.4 for 9.4 at 32 of 8192
    const bool two = !kFull && g.per > 2 * kThinWaves && g.per <= 8 * kThinWaves;
    if (mt == 1 && two)
      thin_kernel<1, 1, kFull ? 1 : 2, kMode, kFull><<<grid, threads, 0, s>>>(g);
    else if (mt == 1)
      thin_kernel<1, 1, 1, kMode, kFull><<<grid, threads, 0, s>>>(g);
    else if (mt == 2)
      thin_kernel<2, 1, 1, kMode, kFull><<<grid, threads, 0, s>>>(g);
    else if (mt == 3)
      thin_kernel<3, 1, 1, kMode, kFull><<<grid, threads, 0, s>>>(g);
    else
      thin_kernel<4, 1, 1, kMode, kFull><<<grid, threads, 0, s>>>(g);
  } else if (p.kernel == kSmall) {
    thin_kernel<4, 2, 1, kMode, kFull><<<grid, 64 * kThinWaves, 0, s>>>(g);
  } else if (p.kernel == kSlim) {
    if (mt <= 2)
      slim_kernel<2, 4, kMode, kFull><<<grid, 256, 0, s>>>(g);
    else if (mt == 3)
      slim_kernel<3, 4, kMode, kFull><<<grid, 256, 0, s>>>(g);
    else
      slim_kernel<4, 4, kMode, kFull><<<grid, 256, 0, s>>>(g);
  } else if constexpr (kFull) {  // 16 bits an operand do not leave registers for more
    tile_kernel<128, 128, 2, 2, 2, 2, kMode, kFull><<<tiles, 256, 0, s>>>(g);
  } else if (p.kernel == kTile128) {
    tile_kernel<128, 128, 4, 2, 2, 4, kMode, kFull><<<tiles, 512, 0, s>>>(g);
  } else if (p.kernel == kTile256x128) {
    tile_kernel<256, 128, 4, 2, 2, 3, kMode, kFull><<<tiles, 512, 0, s>>>(g);
  } else {
    tile_kernel<256, 256, 2, 4, 3, 2, kMode, kFull><<<tiles, 512, 0, s>>>(g);
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
               int64_t row_stride, int64_t block_stride, int scale_type, int64_t K) {
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
  if ((st = check_side("a", a, a_pitch, a_scales, a_row_stride, a_block_stride, scale_type, K)))
    return st;
  if ((st = check_side("b", b, b_pitch, b_scales, b_row_stride, b_block_stride, scale_type, K)))
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
  g.tiles_a = (int32_t)nl2k::ceil_div(M, p.bm);
  g.tiles_b = (int32_t)nl2k::ceil_div(N, p.bn);
  g.tiles = (int32_t)(p.blocks * p.parts);
  const bool full = out_dtype == kF32;
  if (scale_type == kScaleE8M0)
    return full ? launch<kHardware, true>(g, p, stream) : launch<kHardware, false>(g, p, stream);
  if (b_tiles)
    return full ? launch<kTiles, true>(g, p, stream) : launch<kTiles, false>(g, p, stream);
  return full ? launch<kRows, true>(g, p, stream) : launch<kRows, false>(g, p, stream);
}

namespace {

// Where a layer's matrices lie in scratch: codes, then scales, each from a multiple of 256 bytes on.
struct Place {
  size_t codes, scales;
  int64_t pitch, row, block;  // of codes in bytes, of scales in numbers
};

// For M rows of x.  Tiles read 128 bytes of a row at a time: rows from multiples of 128 on are a line
// each, 4096 x 4096 x 2050 with 32-bit scales 40.3 us for 46.0, 1000 x 1111 x 2050 14.9 for 16.1; few
// rows are read as they come, 3 x 5000 x 5000 9.0 us for 10.7 (5120 bytes apart).
struct Scratch {
  const int64_t unit;
  size_t bytes = 0;
  explicit Scratch(int64_t M) : unit(M > 64 ? 128 : 16) {}
  int64_t pitch(int64_t n) const { return nl2k::ceil_div(n, unit) * unit; }
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
  // of rows' blocks, scales blocks first
  Place rows(int64_t m, int64_t k, int scale_type) {
    Place p{};
    p.pitch = pitch(k);
    p.codes = take((size_t)m * p.pitch);
    p.scales = take((size_t)nl2k::ceil_div(k, kBlock) * m * scale_bytes(scale_type));
    p.row = 1, p.block = m;
    return p;
  }
};

// What the forward keeps: x^T [K, M] for dw, w^T [K, N] and w's scales for dx.
struct Kept {
  Place xt, wt;
  size_t bytes;
};
Kept kept_layout(int64_t M, int64_t N, int64_t K, int scale_type, bool dx, bool dw) {
  Scratch s(M);
  Kept k{};
  if (dw) k.xt = s.rows(K, M, scale_type);
  if (dx) {
    k.wt.pitch = s.pitch(N);
    k.wt.codes = s.take((size_t)K * k.wt.pitch);
    k.wt.scales = s.take((size_t)nl2k::ceil_div(N, kBlock) * nl2k::ceil_div(K, kBlock) *
                         scale_bytes(scale_type));
    k.wt.row = 1, k.wt.block = nl2k::ceil_div(K, kBlock);  // of the transposed matrix's tiles
  }
  k.bytes = s.bytes;
  return k;
}

struct ForwardScratch {
  Place x, w;
  size_t product, bytes;
};
ForwardScratch forward_layout(int64_t M, int64_t N, int64_t K, int scale_type, int x_dtype) {
  Scratch s(M);
  ForwardScratch f{};
  f.x = s.rows(M, K, scale_type);
  f.w.pitch = s.pitch(K);
  f.w.codes = s.take((size_t)N * f.w.pitch);
  f.w.scales = s.take((size_t)nl2k::ceil_div(N, kBlock) * nl2k::ceil_div(K, kBlock) *
                      scale_bytes(scale_type));
  f.w.row = nl2k::ceil_div(K, kBlock), f.w.block = 1;
  f.product = s.take(workspace_of(plan(M, N, K, x_dtype == kF32), M, N));
  f.bytes = s.bytes;
  return f;
}

struct BackwardScratch {
  Place dy, dyt;
  size_t product, bytes;
};
BackwardScratch backward_layout(int64_t M, int64_t N, int64_t K, int scale_type, int x_dtype,
                                int w_dtype) {
  // of what the sizes allow
  const bool dx = !check_sizes(M, K, N), dw = !check_sizes(N, K, M);
  Scratch s(M);
  BackwardScratch b{};
  b.dy = s.rows(M, N, scale_type);
  if (dw) b.dyt = s.rows(N, M, scale_type);
  // one product after the other
  b.product =
      s.take(std::max(dx ? workspace_of(plan(M, K, N, x_dtype == kF32), M, K) : 0,
                      dw ? workspace_of(plan(N, K, M, w_dtype == kF32), N, K) : 0));
  b.bytes = s.bytes;
  return b;
}

// Sizes that the products take which are wanted: each has its own sum, of K, of N or of M numbers.
int check_layer(const char* who, int64_t M, int64_t N, int64_t K, int scale_type, int x_dtype,
                int w_dtype, bool dx, bool dw) {
  if (M < 0 || N < 1 || K < 1)
    return nl2k::fail(NL2K_ERR_SHAPE, "%s: need M >= 0, N, K >= 1 (got %lld, %lld, %lld)", who,
                      (long long)M, (long long)N, (long long)K);
  if (check_sizes(M, N, K) || (dx && check_sizes(M, K, N)) || (dw && M && check_sizes(N, K, M)))
    return nl2k::fail(NL2K_ERR_OVERFLOW, "%s: sizes too large (M=%lld N=%lld K=%lld)", who,
                      (long long)M, (long long)N, (long long)K);
  if (x_dtype < kF32 || x_dtype > kF16 || w_dtype < kF32 || w_dtype > kF16 ||
      (scale_type != kScaleF32 && scale_type != kScaleE8M0))
    return nl2k::fail(NL2K_ERR_VALUE, "%s: types must be 0, 1 or 2, scale_type 0 or 1 (got %d, %d, %d)",
                      who, x_dtype, w_dtype, scale_type);
  return NL2K_SUCCESS;
}

int check_scratch(const char* who, const char* name, const void* p, size_t have, size_t need) {
  if (need && (!p || have < need))
    return nl2k::fail(NL2K_ERR_WORKSPACE, "%s: %s of %zu bytes is needed (got %zu)", who, name, need,
                      have);
  if (reinterpret_cast<uintptr_t>(p) % 256)
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: %s must be aligned to 256 bytes", who, name);
  return NL2K_SUCCESS;
}

}  // namespace

extern "C" size_t block_linear_kept_bytes(int64_t M, int64_t N, int64_t K, int scale_type,
                                          int want_dx, int want_dw, int have_codes) {
  if (check_layer("block_linear_kept_bytes", M, N, K, scale_type, 0, 0, want_dx, want_dw) || M == 0)
    return 0;
  return kept_layout(M, N, K, scale_type, want_dx && !have_codes, want_dw).bytes;
}

extern "C" size_t block_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int scale_type,
                                               int x_dtype, int w_dtype, int backward) {
  if (check_layer("block_linear_workspace_bytes", M, N, K, scale_type, x_dtype, w_dtype, false, false) ||
      M == 0)
    return 0;
  return backward ? backward_layout(M, N, K, scale_type, x_dtype, w_dtype).bytes
                  : forward_layout(M, N, K, scale_type, x_dtype).bytes;
}

extern "C" int block_linear_forward(const void* x, int x_dtype, int64_t x_stride, const void* w,
                                    int w_dtype, int64_t w_stride, const void* w_codes,
                                    int64_t w_pitch, const void* w_scales, int64_t w_row_stride,
                                    int64_t w_block_stride, int scale_type, int want_dx,
                                    int want_dw, void* y, void* kept, int64_t M, int64_t N,
                                    int64_t K, void* workspace, size_t workspace_bytes,
                                    hipStream_t stream) {
  const char* who = "block_linear_forward";
  int st = check_layer(who, M, N, K, scale_type, x_dtype, w_dtype, want_dx, want_dw);
  if (st) return st;
  if (M == 0) return nl2k::succeed();
  if (!x || !y || (!w && !w_codes) || !w_codes != !w_scales)
    return nl2k::fail(NL2K_ERR_NULL, "%s: x, y and w, or its codes and scales, are required", who);
  const ForwardScratch f = forward_layout(M, N, K, scale_type, x_dtype);
  const bool keep_w = want_dx && !w_codes;
  const Kept k = kept_layout(M, N, K, scale_type, keep_w, want_dw);
  if ((st = check_scratch(who, "a workspace", workspace, workspace_bytes, f.bytes))) return st;
  if ((st = check_scratch(who, "kept", kept, kept ? k.bytes : 0, k.bytes))) return st;
  char* ws = static_cast<char*>(workspace);
  char* to = static_cast<char*>(kept);
  st = nl2k::quant::run(who, x, x_dtype, x_stride, ws + f.x.codes, f.x.pitch, ws + f.x.scales,
                        want_dw ? to + k.xt.codes : nullptr, k.xt.pitch,
                        want_dw ? to + k.xt.scales : nullptr, scale_type, M, K, false, stream);
  if (st) return st;
  if (!w_codes) {
    void* scales = keep_w ? to + k.wt.scales : ws + f.w.scales;
    st = nl2k::quant::run(who, w, w_dtype, w_stride, ws + f.w.codes, f.w.pitch, scales,
                          keep_w ? to + k.wt.codes : nullptr, k.wt.pitch, nullptr, scale_type, N, K,
                          true, stream);
    if (st) return st;
    w_codes = ws + f.w.codes, w_pitch = f.w.pitch;
    w_scales = scales, w_row_stride = f.w.row, w_block_stride = f.w.block;
  }
  return block_matmul(ws + f.x.codes, f.x.pitch, ws + f.x.scales, f.x.row, f.x.block, 0, w_codes,
                      w_pitch, w_scales, w_row_stride, w_block_stride, 1, scale_type, y, x_dtype, M,
                      N, K, ws + f.product, f.bytes - f.product, stream);
}

extern "C" int block_linear_backward(const void* dy, int x_dtype, int64_t dy_stride,
                                     const void* w_codes_t, int64_t w_pitch_t,
                                     const void* w_scales_t, int64_t w_row_stride_t,
                                     int64_t w_block_stride_t, int scale_type, const void* kept,
                                     void* dx, void* dw, int w_dtype, int64_t M, int64_t N,
                                     int64_t K, void* workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
  const char* who = "block_linear_backward";
  int st = check_layer(who, M, N, K, scale_type, x_dtype, w_dtype, dx, dw);
  if (st) return st;
  if (M == 0 || (!dx && !dw)) return nl2k::succeed();
  const bool kept_w = dx && !w_codes_t;
  if (!dy || !w_codes_t != !w_scales_t || ((kept_w || dw) && !kept))
    return nl2k::fail(NL2K_ERR_NULL, "%s: dy, and what the forward kept, are required", who);
  const BackwardScratch b = backward_layout(M, N, K, scale_type, x_dtype, w_dtype);
  const Kept k = kept_layout(M, N, K, scale_type, kept_w, dw != nullptr);
  if ((st = check_scratch(who, "a workspace", workspace, workspace_bytes, b.bytes))) return st;
  if ((st = check_scratch(who, "kept", kept, k.bytes, k.bytes))) return st;
  char* ws = static_cast<char*>(workspace);
  const char* from = static_cast<const char*>(kept);
  st = nl2k::quant::run(who, dy, x_dtype, dy_stride, ws + b.dy.codes, b.dy.pitch, ws + b.dy.scales,
                        dw ? ws + b.dyt.codes : nullptr, b.dyt.pitch,
                        dw ? ws + b.dyt.scales : nullptr, scale_type, M, N, false, stream);
  if (st) return st;
  if (dw) {
    st = block_matmul(ws + b.dyt.codes, b.dyt.pitch, ws + b.dyt.scales, b.dyt.row, b.dyt.block, 0,
                      from + k.xt.codes, k.xt.pitch, from + k.xt.scales, k.xt.row, k.xt.block, 0,
                      scale_type, dw, w_dtype, N, K, M, ws + b.product, b.bytes - b.product, stream);
    if (st) return st;
  }
  if (!dx) return NL2K_SUCCESS;
  if (kept_w) {
    w_codes_t = from + k.wt.codes, w_pitch_t = k.wt.pitch;
    w_scales_t = from + k.wt.scales, w_row_stride_t = k.wt.row, w_block_stride_t = k.wt.block;
  }
  return block_matmul(ws + b.dy.codes, b.dy.pitch, ws + b.dy.scales, b.dy.row, b.dy.block, 0,
                      w_codes_t, w_pitch_t, w_scales_t, w_row_stride_t, w_block_stride_t, 1,
                      scale_type, dx, x_dtype, M, K, N, ws + b.product, b.bytes - b.product, stream);
}

extern "C" const char* block_matmul_last_error(void) { return nl2k::error_slot().text; }
