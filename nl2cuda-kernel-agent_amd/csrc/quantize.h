// Matrices quantised to e4m3, rows' blocks or tiles', in one direction or both: what block_quant.h
// describes.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "e4m3.h"

namespace nl2k {
namespace quant {

using namespace nl2k::e4m3;

struct Args {
  const void* x;
  uint8_t* codes;
  uint8_t* codes_t;
  void* scales;
  void* scales_t;
  int64_t stride, pitch, pitch_t;
  int32_t M, K;
  uint32_t blocks_k;  // ceil(K / 128)
};

// 16 P rows by 128 columns a workgroup: 16 lanes hold a row, in windows of eight numbers, of each of
// P rows next to each other, so that a lane has P codes of a column, which lie next to each other in
// the transposed matrix.  One read serves both directions.
//
// Bound by memory: 8192 x 8192 bfloat16 in tiles, both ways, 53.5 us (5.0 TB/s, as a large copy),
// 4096 x 4096 in rows 14.1.  Of that, a column's scale by one thread instead of by all that hold the
// column is 17.1 -> 15.6, and the order of the transposed codes in LDS 15.6 -> 14.1; 512 threads of
// four rows each took 21.0.
template <class T, int kType, bool kTiles, bool kT, int P>
__global__ __launch_bounds__(256) void quantize_kernel(Args a) {
  static_assert(P == 8 || (!kT && !kTiles), "a block of the other direction lies in one workgroup");
  constexpr int kPitch = 128 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t turned[kT ? 128 * kPitch : 16];
  __shared__ __attribute__((aligned(16))) float red[kT && !kTiles ? 4 * 128 : 4];
  const uint32_t kb = blockIdx.x % a.blocks_k, mb = blockIdx.x / a.blocks_k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = threadIdx.x >> 4, piece = threadIdx.x & 15;
  const int row0 = group * P;                       // of this lane, in the workgroup
  const int64_t m0 = (int64_t)mb * (16 * P) + row0;  // and in the matrix
  const int k = (int)kb * 128 + piece * 8;
  const auto* x = static_cast<const typename Elem<T>::type*>(a.x);

  Raw<T> raw[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    raw[p] = load8<T>(x + (m0 + p) * a.stride + k, m0 + p < a.M ? a.K - k : 0);

  float top[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float v[8];
    values<T>(raw[p], v);
    top[p] = magnitude(v);
  }
  Scale s[P];
  if constexpr (kTiles) {
    float t = top[0];
#pragma unroll
    for (int p = 1; p < P; ++p) t = fmaxf(t, top[p]);
    t = nl2k::wave_max_dpp(t);
    if (lane == 0) red[wave] = t;
    __syncthreads();
    s[0] = scale_of<kType>(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
#pragma unroll
    for (int p = 1; p < P; ++p) s[p] = s[0];
    if (threadIdx.x == 0) keep<kType>(a.scales, (int64_t)mb * a.blocks_k + kb, s[0].kept);
  } else {
    uint32_t mine = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      s[p] = scale_of<kType>(nl2k::row16_max_dpp(top[p]));
      mine = piece == p ? s[p].kept : mine;
    }
    if (piece < P && m0 + piece < a.M)
      keep<kType>(a.scales, (int64_t)kb * a.M + m0 + piece, mine);
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float v[8];
    values<T>(raw[p], v);
    if (m0 + p < a.M && k < (a.K + 15) / 16 * 16)
      *reinterpret_cast<u32x2*>(a.codes + (m0 + p) * a.pitch + k) = pack8(v, s[p].inverse);
  }
  if constexpr (kT) {
    float inverse[8];
    if constexpr (kTiles) {
#pragma unroll
      for (int e = 0; e < 8; ++e) inverse[e] = s[0].inverse;
    } else {
      float col[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) col[e] = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float v[8];
        values<T>(raw[p], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) col[e] = fmaxf(col[e], fabsf(v[e]));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        col[e] = fmaxf(col[e], __shfl_xor(col[e], 16, 64));
        col[e] = fmaxf(col[e], __shfl_xor(col[e], 32, 64));
      }
      if (lane < 16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) red[wave * 128 + piece * 8 + e] = col[e];
      }
      __syncthreads();
      const int c = threadIdx.x;
      if (c < 128) {
        const Scale t = scale_of<kType>(
            fmaxf(fmaxf(red[c], red[128 + c]), fmaxf(red[256 + c], red[384 + c])));
        const int64_t col = (int64_t)kb * 128 + c;
        if (col < a.K) keep<kType>(a.scales_t, (int64_t)mb * a.K + col, t.kept);
        red[c] = t.inverse;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) inverse[e] = red[piece * 8 + e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        float w[8];
        values<T>(raw[p], w);
        v[p] = w[e];
      }
      // the 16-byte pieces of a column permuted, so that 64 lanes write to all banks
      *reinterpret_cast<u32x2*>(turned + (piece * 8 + e) * kPitch +
                                (((row0 >> 4) ^ (piece >> 1)) * 16 + (row0 & 8))) =
          pack8(v, inverse[e]);
    }
    __syncthreads();
    const int64_t t0 = (int64_t)mb * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = i * 32 + (threadIdx.x >> 3), at = (threadIdx.x & 7) * 16;
      const int64_t kk = (int64_t)kb * 128 + c;
      if (kk < a.K && t0 + at < (a.M + 15) / 16 * 16)
        *reinterpret_cast<u32x4*>(a.codes_t + kk * a.pitch_t + t0 + at) =
            *reinterpret_cast<const u32x4*>(turned + c * kPitch + (at ^ ((c >> 4) * 16)));
    }
  }
}

template <class T, int kType>
inline int launch(const Args& a, bool tiles, hipStream_t stream) {
  const bool t = a.codes_t != nullptr;
  // few rows: a workgroup takes 16 of them, so that more CUs have work.  bfloat16 rows of 4096:
  // 64 rows 2.1 us against 3.3 with 128 a workgroup, 2048 6.0 against 7.2, 4096 10.3 against 10.8,
  // 8192 (2048 workgroups of 128 rows) 20.7 against 20.5.
  const bool few = !tiles && !t && nl2k::ceil_div(a.M, 128) * a.blocks_k < 2048;
  const int64_t blocks = nl2k::ceil_div(a.M, few ? 16 : 128) * a.blocks_k;
  if (blocks > nl2k::max_blocks(256))
    return nl2k::fail(NL2K_ERR_OVERFLOW, "block_quant: more blocks than a launch has (%lld)",
                      (long long)blocks);
  const dim3 grid((uint32_t)blocks);
  if (tiles && t)
    quantize_kernel<T, kType, true, true, 8><<<grid, 256, 0, stream>>>(a);
  else if (tiles)
    quantize_kernel<T, kType, true, false, 8><<<grid, 256, 0, stream>>>(a);
  else if (t)
    quantize_kernel<T, kType, false, true, 8><<<grid, 256, 0, stream>>>(a);
  else if (few)
    quantize_kernel<T, kType, false, false, 1><<<grid, 256, 0, stream>>>(a);
  else
    quantize_kernel<T, kType, false, false, 8><<<grid, 256, 0, stream>>>(a);
  return nl2k::check_launch("block_quant");
}

inline int run(const char* who, const void* x, int dtype, int64_t stride, void* codes, int64_t pitch,
        void* scales, void* codes_t, int64_t pitch_t, void* scales_t, int scale_type, int64_t M,
        int64_t K, bool tiles, hipStream_t stream) {
  if (M < 0 || K < 1)
    return nl2k::fail(NL2K_ERR_SHAPE, "%s: need M >= 0 and K >= 1 (got M=%lld K=%lld)", who,
                      (long long)M, (long long)K);
  if (M > INT32_MAX - 128 || K > INT32_MAX - 128)
    return nl2k::fail(NL2K_ERR_OVERFLOW, "%s: sizes too large (M=%lld K=%lld)", who, (long long)M,
                      (long long)K);
  if (dtype < kF32 || dtype > kF16)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: dtype must be 0, 1 or 2 (got %d)", who, dtype);
  if (scale_type != kScaleF32 && scale_type != kScaleE8M0)
    return nl2k::fail(NL2K_ERR_VALUE, "%s: scale_type must be 0 or 1 (got %d)", who, scale_type);
  if (M == 0) return nl2k::succeed();
  // strides that 64-bit offsets hold
  if (stride < 0 || (M > 1 && stride > INT64_MAX / 8 / M) || pitch < K || pitch % 16 ||
      pitch > INT64_MAX / 8 / M)
    return nl2k::fail(NL2K_ERR_SHAPE,
                      "%s: need stride >= 0 and a pitch of codes >= K, a multiple of 16 (got %lld, "
                      "%lld)", who, (long long)stride, (long long)pitch);
  if (codes_t && (pitch_t < M || pitch_t % 16 || pitch_t > INT64_MAX / 8 / K))
    return nl2k::fail(NL2K_ERR_SHAPE,
                      "%s: the pitch of transposed codes must be >= M, a multiple of 16 (got %lld)",
                      who, (long long)pitch_t);
  if (!x || !codes || !scales || (codes_t && !tiles && !scales_t))
    return nl2k::fail(NL2K_ERR_NULL, "%s: x, codes and scales are required", who);
  if (reinterpret_cast<uintptr_t>(x) % bytes_of(dtype) ||
      reinterpret_cast<uintptr_t>(scales) % scale_bytes(scale_type) ||
      reinterpret_cast<uintptr_t>(scales_t) % scale_bytes(scale_type))
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: x and scales must be aligned to their type", who);
  if (!nl2k::aligned16(codes) || !nl2k::aligned16(codes_t))
    return nl2k::fail(NL2K_ERR_ALIGN, "%s: codes must be aligned to 16 bytes", who);
  const Args a{x,      static_cast<uint8_t*>(codes), static_cast<uint8_t*>(codes_t),
               scales, scales_t,                     M > 1 ? stride : 0,
               pitch,  pitch_t,                      (int32_t)M,
               (int32_t)K, (uint32_t)nl2k::ceil_div(K, kBlock)};
  const bool wide = scale_type == kScaleF32;
  switch (dtype) {
    case kF32:
      return wide ? launch<float, kScaleF32>(a, tiles, stream)
                  : launch<float, kScaleE8M0>(a, tiles, stream);
    case kBF16:
      return wide ? launch<bf16_t, kScaleF32>(a, tiles, stream)
                  : launch<bf16_t, kScaleE8M0>(a, tiles, stream);
    default:
      return wide ? launch<f16_t, kScaleF32>(a, tiles, stream)
                  : launch<f16_t, kScaleE8M0>(a, tiles, stream);
  }
}

}  // namespace quant
}  // namespace nl2k
