// A row's int8 codes and scale, as every kernel that quantises rows makes them.
#pragma once

#include "linear.h"

namespace mi355 {

// 8 values of 16 bits
template <typename E>
__device__ __forceinline__ void unpack_row8(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = E::ld(static_cast<uint16_t>(w[k]));
    f[2 * k + 1] = E::ld(static_cast<uint16_t>(w[k] >> 16));
  }
}
// Columns i .. i + 7 of a row: 16-byte loads when VEC (i a multiple of 8), else those
// below `cols` one by one and zeros.
template <typename E, bool VEC>
__device__ __forceinline__ void row8(const typename E::T* p, int64_t i, int64_t cols, float (&f)[8]) {
  if constexpr (VEC && sizeof(typename E::T) == 2) {
    unpack_row8<E>(*reinterpret_cast<const uint4*>(p + i), f);
  } else if constexpr (VEC) {
    const float4 a = reinterpret_cast<const float4*>(p + i)[0], b = reinterpret_cast<const float4*>(p + i)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = i + k < cols ? E::ld(p[i + k]) : 0.f;
  }
}

// |v| as bits: they order as the values do, a NaN above infinity
__device__ __forceinline__ uint32_t top8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t u = __float_as_uint(f[k]) & 0x7fffffffu;
    m = u > m ? u : m;
  }
  return m;
}
__device__ __forceinline__ uint32_t wave_top(uint32_t m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t u = static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o, 64));
    m = u > m ? u : m;
  }
  return m;
}
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float a = __uint_as_float(top);
  return (a < 1e-10f ? 1e-10f : a) * (1.0f / 127.0f);
}
// 8 codes of a row with scale s: zeros where that is infinite or NaN.  v * (1 / s), added
// to 1.5 * 2^23 in one rounding, leaves its nearest integer (halves to the even one) in the
// sum's low bits.  1 / s is off by 2^-24 of itself, so that is the quotient's integer unless
// the quotient lies within 2^-15 of the middle between two (|q| <= 127: 127 * 2^-23 and
// what the difference's rounding adds): then divisions decide (8 values in a few thousand).
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float s) {
  constexpr float kMagic = 12582912.0f;
  if (!(s < __uint_as_float(0x7f800000u))) return make_uint2(0, 0);
  const float inv = 1.0f / s;
  float m[8], off = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    m[k] = __builtin_fmaf(f[k], inv, kMagic);
    off = fmaxf(off, fabsf(__builtin_fmaf(f[k], inv, kMagic - m[k])));
  }
  if (off > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = __builtin_rintf(f[k] / s) + kMagic;
  }
  auto bytes4 = [&](int k) __attribute__((always_inline)) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(m[k + 1]), __float_as_uint(m[k]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(m[k + 3]), __float_as_uint(m[k + 2]), 0x04000c0cu);
    return lo | hi;
  };
  return make_uint2(bytes4(0), bytes4(4));
}

}  // namespace mi355
