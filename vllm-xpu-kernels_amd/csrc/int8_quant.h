// A row's int8 codes and scale, as every kernel that quantises rows makes them.
#pragma once

#include "linear.h"

namespace mi355 {

// Columns i .. i + 7 of a row: 16-byte loads when VEC (i a multiple of 8), else those
// below `cols` one by one and zeros.
template <typename E, bool VEC>
__device__ __forceinline__ void row8(const typename E::T* p, int64_t i, int64_t cols, float (&f)[8]) {
  if constexpr (VEC && sizeof(typename E::T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = E::ld(static_cast<uint16_t>(w[k]));
      f[2 * k + 1] = E::ld(static_cast<uint16_t>(w[k] >> 16));
    }
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
// The code of v / s.  v * (1 / s) is off by less than 2^-15 (three roundings of a value up
// to 127), so its nearest integer is the quotient's unless it lies that near the middle
// between two: then the division decides (a few of 100000 values).
__device__ __forceinline__ int code_of(float v, float s, float inv) {
  const float t = v * inv;
  float r = __builtin_rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) < 0x1p-14f) r = __builtin_rintf(v / s);
  return static_cast<int>(r);
}
// 8 codes of a row with scale s: zeros where that is infinite or NaN
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float s) {
  uint32_t w[2] = {0, 0};
  if (s < __uint_as_float(0x7f800000u)) {
    const float inv = 1.0f / s;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      w[k >> 2] |= static_cast<uint32_t>(code_of(f[k], s, inv) & 0xff) << (8 * (k & 3));
  }
  return make_uint2(w[0], w[1]);
}

}  // namespace mi355
