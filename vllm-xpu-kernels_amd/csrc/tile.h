// What tile kernels share: copies from global memory straight into LDS, their waits, and
// loops over constants.
#pragma once

#include <stdint.h>

#include <type_traits>

#include <hip/hip_runtime.h>

namespace mi355 {

typedef __attribute__((address_space(3))) void lds_void_t;

__device__ __forceinline__ uint32_t lds_off(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)p));
}
// 16 / 4 bytes per lane from sbase + voff (scalar base, 32-bit lane offset) into
// LDS at lds_base + OFF + 16 (4) lane
// (s_nop: M0 takes one wait state from its write to the copy that reads it)
template <int OFF>
__device__ __forceinline__ void dma16(uint32_t voff, uint64_t sbase, uint32_t lds_base) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds_base), "n"(OFF) : "memory", "m0", "scc");
}
__device__ __forceinline__ void dma4(uint32_t voff, uint64_t sbase, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32)));
  return (hi << 32) | lo;
}
__device__ __forceinline__ uint64_t uniform_ptr(const void* p) {
  return uniform64(reinterpret_cast<uint64_t>(p));
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N < 64, "vmcnt has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// this wave's LDS reads and writes are done, then every wave's
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// f(integral_constant 0), ..., f(integral_constant N - 1)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void for_each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each<N, I + 1>(f);
  }
}

}  // namespace mi355
