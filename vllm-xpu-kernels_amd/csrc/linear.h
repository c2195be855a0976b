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
//
// int8 products.  Sums of 8-bit products are int32 and exact (K < 2^17: 2^17 products
// of -128 reach 2^31), and every kernel takes the same fp32 steps from there, so a result is
// the same whichever kernel, tile or split made it:
//   z[m, n] = fma(float(sum), x_scale[m] * weight_scale[n], bias[n] or 0)  (scaled_sum),
// then the activation, a product with the gated factor and a sum with the residual, each
// rounded once (times, plus: the compiler would contract such a pair where both
// meet in one block, in some kernels and not in others).
#pragma once

#include <type_traits>

#include "mfma16.h"

namespace mi355 {

typedef mi355moe_linear_args LinArgs;
typedef int lin_i32x4 __attribute__((ext_vector_type(4)));

// operands of a kernel; K_FP8_EXACT: e4m3 with the bf16 MFMA's sums
enum { K_BF16 = 0, K_F16 = 1, K_FP8 = 2, K_FP8_EXACT = 3, K_I8 = 4 };
constexpr __host__ __device__ bool kind_fp8(int kind) { return kind == K_FP8 || kind == K_FP8_EXACT; }
constexpr __host__ __device__ int kind_bytes(int kind) { return kind == K_BF16 || kind == K_F16 ? 2 : 1; }
inline int kind_of(const LinArgs& a) {
  return a.x_dtype == MI355MOE_FP8E4M3 ? K_FP8 : a.x_dtype == MI355MOE_I8 ? K_I8
         : a.x_dtype == MI355MOE_F16 ? K_F16 : K_BF16;
}
// a kernel's sums: int32 of int8 products, else float
template <int KIND, int N>
struct SumVec { typedef float T __attribute__((ext_vector_type(N))); };
template <int N>
struct SumVec<K_I8, N> { typedef int T __attribute__((ext_vector_type(N))); };

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

// K step of 16 bytes per lane: 16 rows x 16 columns (32 16-bit or 64 8-bit k) ...
template <int KIND>
__device__ __forceinline__ typename SumVec<KIND, 4>::T mfma_16x16(uint4 a, uint4 b,
                                                                  typename SumVec<KIND, 4>::T c) {
  if constexpr (KIND == K_I8)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(lin_i32x4, a),
                                                 __builtin_bit_cast(lin_i32x4, b), c, 0, 0, 0);
  else return mfma16_16x16x32<KIND == K_F16>(a, b, c);
}
// ... and 32 x 32 (16 16-bit or 32 8-bit k)
template <int KIND>
__device__ __forceinline__ typename SumVec<KIND, 16>::T mfma_32x32(uint4 a, uint4 b,
                                                                   typename SumVec<KIND, 16>::T c) {
  if constexpr (KIND == K_I8)
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(lin_i32x4, a),
                                                 __builtin_bit_cast(lin_i32x4, b), c, 0, 0, 0);
  else return mfma16_32x32x16<KIND == K_F16>(a, b, c);
}

// int8: row m's and weight row n's scales
__device__ __forceinline__ float x_scale_of(const LinArgs& a, int64_t m) {
  return a.x_scale[m * a.x_scale_row];
}
__device__ __forceinline__ float w_scale_of(const LinArgs& a, int64_t n) {
  return a.weight_scale[n * a.weight_scale_row];
}

// ... and its sum, scaled and biased in one rounding (bias: 0 where there is none)
__device__ __forceinline__ float scaled_sum(int sum, float x_scale, float weight_scale, float bias) {
  return __builtin_fmaf(static_cast<float>(sum), x_scale * weight_scale, bias);
}
// the products and sums of an epilogue, never contracted
__device__ __forceinline__ float times(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
__device__ __forceinline__ float plus(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
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
    return times(r, r);
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

// One output: z and, for gated activations, the factor u, both without bias (BIASED: with it).
// KEEP: z and u with their biases are kept too (a.z).
template <bool KEEP = false, bool BIASED = false>
__device__ __forceinline__ float lin_value(const LinArgs& a, int64_t m, int64_t n, float z,
                                           float u) {
  if (!BIASED && a.bias) z += ld_any(a.bias, a.bias_dtype, n);
  float v[1] = {z};
  lin_act(a.activation, v);
  float y = v[0];
  if (lin_gated(a.activation)) {
    if (!BIASED && a.bias) u += ld_any(a.bias, a.bias_dtype, a.N + n);
    y = times(y, u);
  }
  if constexpr (KEEP) {
    a.z[m * 2 * a.N + n] = z;
    a.z[(m * 2 + 1) * a.N + n] = u;
  }
  if (a.residual) y = plus(y, ld_any(a.residual, a.residual_dtype, m * a.ldr + n));
  return y;
}
// The same of an int8 product's sums.
__device__ __forceinline__ float lin_value_i32(const LinArgs& a, int64_t m, int64_t n, float x_scale,
                                               int z, int u) {
  auto scaled = [&](int sum, int64_t row) __attribute__((always_inline)) {
    return scaled_sum(sum, x_scale, w_scale_of(a, row), a.bias ? ld_any(a.bias, a.bias_dtype, row) : 0.f);
  };
  return lin_value<false, true>(a, m, n, scaled(z, n), lin_gated(a.activation) ? scaled(u, a.N + n) : 0.f);
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

// 8 floats to p, by 16 bytes where `vec`
__device__ __forceinline__ void st8_f32(float* p, const float (&y)[8], bool vec) {
  if (vec) {
    float4* o = reinterpret_cast<float4*>(p);
    o[0] = make_float4(y[0], y[1], y[2], y[3]);
    o[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] = y[k];
  }
}
// Outputs n .. n + 7 (those below N) of row m from their sums z and, for gated
// activations, u (BIASED: with their biases).  vec: out's rows start at multiples of 16 bytes.
// early: res holds the 8 (16-bit) residuals, loaded before.
template <bool KEEP = false, bool BIASED = false>
__device__ __forceinline__ void lin_store8(const LinArgs& a, int64_t m, int64_t n, const float* zp,
                                           const float* up, bool vec, bool early = false,
                                           uint4 res = uint4{}) {
  if (n + 8 > a.N) {
    for (int k = 0; k < 8 && n + k < a.N; ++k)
      st_any(a.out, a.out_dtype, m * a.ldo + n + k, lin_value<KEEP, BIASED>(a, m, n + k, zp[k], up[k]));
    return;
  }
  const bool gated = lin_gated(a.activation);
  float y[8], t[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = zp[k];
  if (!BIASED && a.bias) {
    ld8_any(a.bias, a.bias_dtype, n, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] += t[k];
  }
  if constexpr (KEEP) st8_f32(a.z + m * 2 * a.N + n, y, (a.N & 3) == 0);
  lin_act(a.activation, y);
  if (gated) {
    float u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = up[k];
    if (!BIASED && a.bias) {
      ld8_any(a.bias, a.bias_dtype, a.N + n, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] += t[k];
    }
    if constexpr (KEEP) st8_f32(a.z + (m * 2 + 1) * a.N + n, u, (a.N & 3) == 0);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = times(y[k], u[k]);
  }
  if (early) {
    unpack8(res, a.residual_dtype, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = plus(y[k], t[k]);
  } else if (a.residual) {
    ld8_any(a.residual, a.residual_dtype, m * a.ldr + n, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = plus(y[k], t[k]);
  }
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) st_any(a.out, a.out_dtype, m * a.ldo + n + k, y[k]);
  } else if (a.out_dtype == MI355MOE_F32) {
    st8_f32(static_cast<float*>(a.out) + m * a.ldo + n, y, true);
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

// The same from the sums of int8 products.
__device__ __forceinline__ void lin_store8_i32(const LinArgs& a, int64_t m, int64_t n, const int* zp,
                                               const int* up, bool vec) {
  const float xs = x_scale_of(a, m);
  float z[8], u[8];
  auto scaled = [&](const int* sums, int64_t row, float (&o)[8]) __attribute__((always_inline)) {
    float b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = 0.f;
    if (a.bias && n + 8 <= a.N) {
      ld8_any(a.bias, a.bias_dtype, row, b);
    } else if (a.bias) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < a.N) b[k] = ld_any(a.bias, a.bias_dtype, row + k);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      o[k] = scaled_sum(sums[k], xs, w_scale_of(a, n + k < a.N ? row + k : row), b[k]);
  };
  scaled(zp, n, z);
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = 0.f;
  if (lin_gated(a.activation)) scaled(up, a.N + n, u);
  lin_store8<false, true>(a, m, n, z, u, vec);
}

// 16 bytes from column byte c of a row of `bytes` bytes, from any address;
// zeros past its end and for rows that do not exist.  (A piece that the row's end cuts is
// loaded byte by byte, each load waited for: that chain, not the way through registers, is
// what kernels on such rows spend most of their time on.)
typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ uint4 row16(const uint8_t* row, bool ok, int64_t c, int64_t bytes) {
  if (!ok || c >= bytes) return make_uint4(0, 0, 0, 0);
  if (c + 16 <= bytes) {
    const any_u32x4 v = *reinterpret_cast<const any_u32x4*>(row + c);
    return make_uint4(v.x, v.y, v.z, v.w);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 15; ++k)
    if (c + k < bytes) w[k >> 2] |= static_cast<uint32_t>(row[c + k]) << (8 * (k & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// codes and scales of 16- or 32-bit rows (int8_quant.hip); pad: zeros behind each row's codes up
// to a multiple of 16
int launch_int8_quant(int dtype, const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                      int64_t scale_row, int64_t rows, int64_t cols, hipStream_t st, bool pad = false);
// rows of `bytes` bytes, ld bytes apart, to rows of a multiple of 16 with zeros behind them
// (linear.hip)
int launch_pack_rows(const void* src, int64_t ld, int64_t bytes, void* dst, int64_t rows, hipStream_t st);
// the sum of a split product's partial sums, in their order, then the epilogue (linear.hip)
int launch_linear_finish(const LinArgs& a, const void* part, int splits, hipStream_t st);
// few rows of x (linear_skinny.hip), any alignment; tile: the tiles can take them too
bool linear_skinny_takes(const LinArgs& a, bool tile);
int launch_linear_skinny(const LinArgs& a, hipStream_t st);
// 16-bit rows of x (a.weight_dtype int8) that it quantises itself
bool linear_skinny_quantises(const LinArgs& a);
// more rows (linear_tile.hip).  a0: the call; a: the same, or with a split K the
// product of all weight rows into fp32 partial sums [splits][M][rows]
bool linear_tile_supported(const LinArgs& a);
int linear_tile_splits(const LinArgs& a);
int launch_linear_tile(const LinArgs& a0, const LinArgs& a, hipStream_t st);
// the same for int8 operands and for kept sums (linear_gemm.hip)
int linear_gemm_splits(const LinArgs& a);
int launch_linear_gemm(const LinArgs& a0, const LinArgs& a, hipStream_t st);

}  // namespace mi355
