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
// 2^-14 below does not), 1.5e-5 of a result's size for normal operands: 130
// times less than half a step of bf16.  Kernels that are bound by the matrix
// cores use it for 16-bit outputs; float32 outputs, and the kernels that
// stream weights, convert the codes to bf16 (exact) and use the 16-bit MFMA,
// whose sums have fp32's precision (1e-7).
#pragma once

#include "mfma16.h"

namespace mi355 {

typedef mi355moe_linear_args LinArgs;

__host__ __device__ constexpr bool lin_gated(int act) {
  return act >= MI355MOE_LINEAR_SILU_AND_MUL;
}

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

// f of the activation (gated ones: f of the gate).  SiLU with the hardware
// exp2 and reciprocal (about 1 ulp each): z -> -inf gives z * rcp(inf) = -0,
// z -> +inf gives z.
__device__ __forceinline__ float lin_act(int act, float z) {
  switch (act) {
    case MI355MOE_LINEAR_SILU:
    case MI355MOE_LINEAR_SILU_AND_MUL:
      return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z * 1.4426950408889634f));
    case MI355MOE_LINEAR_GELU:
    case MI355MOE_LINEAR_GELU_AND_MUL: return gelu_erf(z);
    case MI355MOE_LINEAR_GELU_TANH:
    case MI355MOE_LINEAR_GELU_TANH_AND_MUL: return gelu_tanh(z);
    case MI355MOE_LINEAR_RELU2: {
      const float r = z < 0.f ? 0.f : z;  // keeps NaN
      return r * r;
    }
    default: return z;
  }
}

// One output: z and, for gated activations, the factor u, both without bias.
__device__ __forceinline__ float lin_value(const LinArgs& a, int64_t m, int64_t n, float z,
                                           float u) {
  if (a.bias) z += ld_any(a.bias, a.bias_dtype, n);
  float y = lin_act(a.activation, z);
  if (lin_gated(a.activation)) {
    if (a.bias) u += ld_any(a.bias, a.bias_dtype, a.N + n);
    y *= u;
  }
  if (a.residual) y += ld_any(a.residual, a.residual_dtype, m * a.ldr + n);
  return y;
}

}  // namespace mi355
