// Numbers in 8 bits (OCP e4m3: 448 the largest, no infinity) with a scale for
// each block of 128, and eight numbers of a row at a time: what the norm, the
// quantisers and the product share.
//
//   s = max(a / 448, 2^-126), a the block's largest magnitude; or the least
//       power of two that is no smaller, kept as its exponent (e8m0)
//   q = e4m3(x * fl(1 / s)), to nearest even
//
// |x| fl(1 / s) <= 448 (1 + 2^-22), which rounds to 448, so nothing needs to be
// clamped.  A NaN stays in its own number; an infinity makes its block's scale
// infinite (e8m0: NaN), and with it all that the block stands for NaN.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"

namespace nl2k {
namespace e4m3 {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };          // types of numbers, as the C entries take them
enum { kScaleF32 = 0, kScaleE8M0 = 1 };          // and of scales
constexpr int kBlock = 128;                      // numbers that share a scale

struct bf16_t {};
struct f16_t {};
template <class T>
struct Elem {
  using type = unsigned short;
  static constexpr int bytes = 2;
};
template <>
struct Elem<float> {
  using type = float;
  static constexpr int bytes = 4;
};

inline int bytes_of(int dtype) { return dtype == kF32 ? 4 : 2; }
inline int scale_bytes(int type) { return type == kScaleF32 ? 4 : 1; }

typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

template <class T>
__device__ __forceinline__ float widen(typename Elem<T>::type h) {
  if constexpr (__is_same(T, float))
    return h;
  else if constexpr (__is_same(T, bf16_t))
    return __builtin_bit_cast(float, (uint32_t)h << 16);
  else
    return (float)__builtin_bit_cast(_Float16, h);
}

// To nearest even.
template <class T>
__device__ __forceinline__ typename Elem<T>::type narrow(float v) {
  if constexpr (__is_same(T, float))
    return v;
  else if constexpr (__is_same(T, bf16_t))
    return __builtin_bit_cast(unsigned short, (__bf16)v);
  else
    return __builtin_bit_cast(unsigned short, (_Float16)v);
}

// Eight numbers as they lie in memory, at any alignment of their type.
template <class T>
struct Raw {
  u16x8 h;
};
template <>
struct Raw<float> {
  f32x4 a, b;
};

// `count` >= 8 numbers from p on, or the first `count` and zeros.
template <class T>
__device__ __forceinline__ Raw<T> load8(const typename Elem<T>::type* p, int count) {
  Raw<T> r;
  if constexpr (__is_same(T, float)) {
    if (count >= 8) {
      r.a = *reinterpret_cast<const f32x4_u*>(p);
      r.b = *reinterpret_cast<const f32x4_u*>(p + 4);
    } else {
      r.a = r.b = zero4();
      if (count > 0) {  // a branch that waves whose rows are whole do not enter
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r.a[e] = e < count ? p[e] : 0.f;
          r.b[e] = e + 4 < count ? p[e + 4] : 0.f;
        }
      }
    }
  } else {
    if (count >= 8) {
      r.h = __builtin_bit_cast(u16x8, (u32x4)*reinterpret_cast<const u32x4_u*>(p));
    } else {
      r.h = u16x8{};
      if (count > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.h[e] = e < count ? p[e] : (unsigned short)0;
      }
    }
  }
  return r;
}

template <class T>
__device__ __forceinline__ void values(const Raw<T>& r, float (&v)[8]) {
  if constexpr (__is_same(T, float)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r.a[e], v[4 + e] = r.b[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widen<T>(r.h[e]);
  }
}

template <class T>
__device__ __forceinline__ void store8(typename Elem<T>::type* p, int count, const float (&v)[8]) {
  if constexpr (__is_same(T, float)) {
    if (count >= 8) {
      *reinterpret_cast<f32x4_u*>(p) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_u*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else if (count > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = v[e];
    }
  } else {
    u16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = narrow<T>(v[e]);
    if (count >= 8) {
      *reinterpret_cast<u32x4_u*>(p) = __builtin_bit_cast(u32x4, h);
    } else if (count > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = h[e];
    }
  }
}

// A block's scale as it is kept (its float, or its exponent), and what its numbers are multiplied
// by.
struct Scale {
  uint32_t kept;
  float inverse;
};

template <int kType>
__device__ __forceinline__ Scale scale_of(float a) {
  if constexpr (kType == kScaleF32) {
    const float s = fmaxf(a / 448.f, 0x1p-126f);
    return Scale{__builtin_bit_cast(uint32_t, s), 1.f / s};
  } else {
    // a = 1.f 2^(e - 127) <= 448 2^k = 1.75 2^(k + 8): k = e - 135, or one more where f > 0.75
    const uint32_t bits = __builtin_bit_cast(uint32_t, a);
    const int e = (int)(bits >> 23);
    const int code = max(e - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), 1);
    if (e == 255) return Scale{255u, 0.f};
    return Scale{(uint32_t)code, __builtin_bit_cast(float, (uint32_t)(254 - code) << 23)};
  }
}

// The largest magnitude; a NaN is passed over.
__device__ __forceinline__ float magnitude(const float (&v)[8]) {
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e]));
  return a;
}

__device__ __forceinline__ u32x2 pack8(const float (&v)[8], float inverse) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inverse, v[4 * i + 1] * inverse, 0, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse, q, true);
    w[i] = (uint32_t)q;
  }
  return w;
}

template <int kType>
__device__ __forceinline__ void keep(void* scales, int64_t at, uint32_t kept) {
  if constexpr (kType == kScaleF32)
    static_cast<uint32_t*>(scales)[at] = kept;
  else
    static_cast<uint8_t*>(scales)[at] = (uint8_t)kept;
}

}  // namespace e4m3
}  // namespace nl2k
