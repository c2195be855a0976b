// Matrix product with bias, activation and residual in its epilogue
// (mi355moe_linear): what its kernels share.
//
//   z[m, n] = sum_k x[m, k] w[n, k] + bias[n]
//   out[m, n] = T(act(z)[m, n] + residual[m, n])
//
// Every kernel takes the weight rows as the MFMA A operand and the rows of x
// as B, so a lane's accumulators are consecutive output columns n of one row m;
// gated activations accumulate the gate's row n and the factor's row N + n in
// the same lane.  Sums, scales, activation and residual are fp32; the output
// is rounded once.
//
// e4m3 products.  The 128-long MFMA adds the products of 8 consecutive k as
// integers of 2^-13 of the largest one's power of two, cut off towards zero
// (measured with single products: one 2^-13 below another of its 8 counts, one
// 2^-14 below does not; the 32-long e4m3 MFMA cuts alike).  Each 8 lose less than
// 7 * 2^-13 of their largest product: 2e-5 of a result's size for normal
// operands, 190 times less than half a step of bf16, 24 times less than fp16's, and
// more of a result whose products cancel.  Converted to bf16 (exact) the
// codes take the 16-bit MFMA, whose sums have fp32's precision (1e-7), at 1.03
// (64 x 4096 x 4096, 16.0 -> 16.5 us) to 1.4 times (8192 x 4096 x 4096, 211 -> 295)
// the time.  Tiles use the e4m3 MFMA for 16-bit outputs and convert for float32
// outputs; the kernels that stream weights (bound by the stream) and the one for any
// alignment always convert.
#pragma once

#include <type_traits>

#include "mfma16.h"

namespace mi355 {

typedef mi355moe_linear_args LinArgs;

__host__ __device__ constexpr bool lin_gated(int act) {
  return act >= MI355MOE_LINEAR_SILU_AND_MUL;
}

// rows of the weight
inline int64_t lin_rows(const LinArgs& a) { return lin_gated(a.activation) ? 2 * a.N : a.N; }

// element i of a float32, bfloat16 or float16 array
__device__ __forceinline__ float ld_any(const void* p, int dtype, int64_t i) {
  if (dtype == MI355MOE_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return dtype == MI355MOE_BF16 ? bf16_to_f32(v) : f16_to_f32(v);
}
__device__ __forceinline__ void st_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == MI355MOE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dtype == MI355MOE_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}

// f of the activation (gated ones: f of the gate).  x sigmoid(k x) with the
// hardware exp2 and reciprocal (about 1 ulp each): a finite x whose exp2
// overflows gives x * rcp(inf) = -0, one whose exp2 vanishes gives x; x = inf
// stays, x = -inf is -inf * 0 = NaN, as x / (1 + exp(-x)) is.  SiLU is k = 1; the tanh form of GELU is
// exactly x sigmoid(2 t), t = sqrt(2/pi) (x + 0.044715 x^3), since (1 + tanh t) / 2
// = sigmoid(2 t); it takes 8 instructions instead of tanhf's 40.
__device__ __forceinline__ float mul_sigmoid(float x, float t) {
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t * -1.4426950408889634f));
}
template <int ACT>
__device__ __forceinline__ float lin_f(float z) {
  if constexpr (ACT == MI355MOE_LINEAR_SILU) return mul_sigmoid(z, z);
  else if constexpr (ACT == MI355MOE_LINEAR_GELU) return gelu_erf(z);
  else if constexpr (ACT == MI355MOE_LINEAR_GELU_TANH)
    return mul_sigmoid(z, 1.5957691216057308f * (z + 0.044715f * (z * z * z)));
  else if constexpr (ACT == MI355MOE_LINEAR_RELU2) {
    const float r = z < 0.f ? 0.f : z;  // keeps NaN
    return r * r;
  } else return z;
}
// f of N values: one (uniform) branch for all
template <int N>
__device__ __forceinline__ void lin_act(int act, float (&y)[N]) {
  auto all = [&](auto a) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = lin_f<decltype(a)::value>(y[k]);
  };
  switch (act) {
    case MI355MOE_LINEAR_SILU:
    case MI355MOE_LINEAR_SILU_AND_MUL:
      all(std::integral_constant<int, MI355MOE_LINEAR_SILU>{});
      break;
    case MI355MOE_LINEAR_GELU:
    case MI355MOE_LINEAR_GELU_AND_MUL:
      all(std::integral_constant<int, MI355MOE_LINEAR_GELU>{});
      break;
    case MI355MOE_LINEAR_GELU_TANH:
    case MI355MOE_LINEAR_GELU_TANH_AND_MUL:
      all(std::integral_constant<int, MI355MOE_LINEAR_GELU_TANH>{});
      break;
    case MI355MOE_LINEAR_RELU2:
      all(std::integral_constant<int, MI355MOE_LINEAR_RELU2>{});
      break;
    default: break;
  }
}

// One output: z and, for gated activations, the factor u, both without bias.
__device__ __forceinline__ float lin_value(const LinArgs& a, int64_t m, int64_t n, float z,
                                           float u) {
  if (a.bias) z += ld_any(a.bias, a.bias_dtype, n);
  float v[1] = {z};
  lin_act(a.activation, v);
  float y = v[0];
  if (lin_gated(a.activation)) {
    if (a.bias) u += ld_any(a.bias, a.bias_dtype, a.N + n);
    y *= u;
  }
  if (a.residual) y += ld_any(a.residual, a.residual_dtype, m * a.ldr + n);
  return y;
}

__device__ __forceinline__ void unpack8(uint4 v, int dtype, float (&f)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  if (dtype == MI355MOE_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack16x2<false>(u[k], f[2 * k], f[2 * k + 1]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack16x2<true>(u[k], f[2 * k], f[2 * k + 1]);
  }
}
// Elements i .. i + 7 of a float32, bfloat16 or float16 array: 16-byte loads
// where the address allows.
__device__ __forceinline__ void ld8_any(const void* p, int dtype, int64_t i, float (&f)[8]) {
  const uint8_t* q = static_cast<const uint8_t*>(p) + i * (dtype == MI355MOE_F32 ? 4 : 2);
  if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
    const uint4 v = *reinterpret_cast<const uint4*>(q);
    if (dtype == MI355MOE_F32) {
      const uint4 w = reinterpret_cast<const uint4*>(q)[1];
      const uint32_t u[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(u[k]);
    } else {
      unpack8(v, dtype, f);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = ld_any(p, dtype, i + k);
  }
}

// Outputs n .. n + 7 (those below N) of row m from their sums z and, for gated
// activations, u.  vec: out's rows start at multiples of 16 bytes.  early: res
// holds the 8 (16-bit) residuals, loaded before.
__device__ __forceinline__ void lin_store8(const LinArgs& a, int64_t m, int64_t n, const float* zp,
                                           const float* up, bool vec, bool early = false,
                                           uint4 res = uint4{}) {
  if (n + 8 > a.N) {
    for (int k = 0; k < 8 && n + k < a.N; ++k)
      st_any(a.out, a.out_dtype, m * a.ldo + n + k, lin_value(a, m, n + k, zp[k], up[k]));
    return;
  }
  const bool gated = lin_gated(a.activation);
  float y[8], t[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = zp[k];
  if (a.bias) {
    ld8_any(a.bias, a.bias_dtype, n, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] += t[k];
  }
  lin_act(a.activation, y);
  if (gated) {
    float u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = up[k];
    if (a.bias) {
      ld8_any(a.bias, a.bias_dtype, a.N + n, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] += t[k];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] *= u[k];
  }
  if (early) {
    unpack8(res, a.residual_dtype, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] += t[k];
  } else if (a.residual) {
    ld8_any(a.residual, a.residual_dtype, m * a.ldr + n, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] += t[k];
  }
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) st_any(a.out, a.out_dtype, m * a.ldo + n + k, y[k]);
  } else if (a.out_dtype == MI355MOE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + m * a.ldo + n);
    o[0] = make_float4(y[0], y[1], y[2], y[3]);
    o[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = a.out_dtype == MI355MOE_BF16 ? pack16x2<false>(y[2 * k], y[2 * k + 1])
                                          : pack16x2<true>(y[2 * k], y[2 * k + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + m * a.ldo + n) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// few rows of x (linear_skinny.hip), any alignment; tile: the tiles can take them too
bool linear_skinny_takes(const LinArgs& a, bool tile);
int launch_linear_skinny(const LinArgs& a, hipStream_t st);
// more rows (linear_tile.hip).  a0: the call; a: the same, or with a split K the
// product of all weight rows into fp32 partial sums [splits][M][rows]
bool linear_tile_supported(const LinArgs& a);
int linear_tile_splits(const LinArgs& a);
int launch_linear_tile(const LinArgs& a0, const LinArgs& a, hipStream_t st);

}  // namespace mi355
