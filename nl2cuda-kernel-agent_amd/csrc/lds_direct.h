// Loads from global memory straight to LDS, counted and waited for by hand, and
// the barriers that go with them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace nl2k {
namespace lds {

// An address that is the same in all lanes, in scalar registers, five issues after whatever
// wrote them.
template <class T>
__device__ __forceinline__ const T* scalar_base(const T* base) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32));
  uint64_t q = hi << 32 | lo;
  asm volatile("s_nop 4" : "+s"(q));
  return reinterpret_cast<const T*>(q);
}

// 16 bytes a lane from global memory straight to LDS: lane n's land at lds + 16 n.
// The count of outstanding loads is waited for by hand (wait_tile): the
// compiler, which does not know which part of LDS a load writes, would have
// every read of LDS wait for all of them.  M0 holds the place in LDS.  A scalar
// register that a vector instruction wrote must not be read by a load within five
// issues, which the compiler does not see to here: `base` comes from
// scalar_base and is moved on by scalar additions alone.
__device__ __forceinline__ void load_lds16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}

// The same with 4 bytes a lane, or one that is widened to 4: lane n's land at lds + 4 n.
template <int kBytes>
__device__ __forceinline__ void load_lds4(const void* base, uint32_t off, uint32_t lds) {
  if constexpr (kBytes == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %2"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
}

// Where a __shared__ array begins, as the loads above take it.
__device__ __forceinline__ uint32_t offset_of(const void* shared) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)shared;
}

// Waits until at most N of this wave's loads are outstanding.
template <int N>
__device__ __forceinline__ void wait_tile() {
  static_assert(N < 64, "the counter has six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0xf70);
}

// Waits until none of its LDS reads are.
__device__ __forceinline__ void wait_reads() { __builtin_amdgcn_s_waitcnt(0xc07f); }

// The barrier alone: what it waits for, wait_tile has waited for.  The compiler may move no
// access across it.
__device__ __forceinline__ void workgroup_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Between what the lanes of a wave write to its part of LDS and read there: LDS keeps a wave's
// accesses in order, so the compiler has to keep them too.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace lds
}  // namespace nl2k
