// Root-mean-square norm of rows with the residual's addition before it and its
// result in the input's type, in e4m3 with a scale per group of columns, or
// both (mi355moe_rms_norm).  Per row, in fp32:
//   h = x + residual,  y = h / sqrt(sum(h^2) / cols + eps) * weight
// and per group of columns of y the scale and codes of the group quantisers
// (per_token_group_fp8_quant's arithmetic; e8m0 scales as the mxfp8 layer's).
//
// One workgroup per row: a pass that sums the squares, a workgroup sum, and a
// pass that reads the row again (from L2) and writes the outputs.
#include "common.h"

namespace mi355 {
namespace {

typedef mi355moe_rms_norm_args NormArgs;

// Elements i .. i + 7 of a row (i a multiple of 8): two or one 16-byte loads
// when VEC, else the elements below `cols` one by one and zeros.
template <typename E, bool VEC>
__device__ __forceinline__ void load8(const void* p, int64_t i, int64_t cols, float (&f)[8]) {
  const typename E::T* q = static_cast<const typename E::T*>(p) + i;
  if constexpr (VEC && sizeof(typename E::T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(q);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = E::ld(static_cast<uint16_t>(w[k]));
      f[2 * k + 1] = E::ld(static_cast<uint16_t>(w[k] >> 16));
    }
  } else if constexpr (VEC) {
    const uint4 a = reinterpret_cast<const uint4*>(q)[0], b = reinterpret_cast<const uint4*>(q)[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = i + k < cols ? E::ld(q[k]) : 0.f;
  }
}
template <typename E, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t i, int64_t cols, const float (&f)[8]) {
  typename E::T* q = static_cast<typename E::T*>(p) + i;
  if constexpr (VEC && sizeof(typename E::T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = static_cast<uint32_t>(E::st(f[2 * k])) |
             (static_cast<uint32_t>(E::st(f[2 * k + 1])) << 16);
    *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if constexpr (VEC) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(f[k]);
    reinterpret_cast<uint4*>(q)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(q)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < cols) q[k] = E::st(f[k]);
  }
}

template <typename E>
__device__ __forceinline__ int64_t row_at(int64_t r, int64_t inner, int64_t outer_stride,
                                          int64_t inner_stride) {
  const int64_t o = inner == 1 ? r * outer_stride
                               : (r / inner) * outer_stride + (r % inner) * inner_stride;
  return o * static_cast<int64_t>(sizeof(typename E::T));
}

// e4m3 code of clamp(v, +-448); a NaN stays one (fminf and fmaxf drop it).
__device__ __forceinline__ float clamp448(float v) {
  const float c = fminf(fmaxf(v, -448.f), 448.f);
  return v == v ? c : v;
}
__device__ __forceinline__ uint32_t e4m3x4_nan(float v0, float v1, float v2, float v3) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(v0), clamp448(v1), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(v2), clamp448(v3), w, true);
  return static_cast<uint32_t>(w);
}

// The group's scale and the lane's 8 codes.  A group is G / 8 consecutive,
// aligned lanes, all of them active (cols % G == 0).
template <bool VEC>
__device__ __forceinline__ void quant8(const NormArgs& a, int64_t r, int64_t i,
                                       const float (&y)[8]) {
  float amax = 1e-10f;
#pragma unroll
  for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(y[k]));
  const int lanes = static_cast<int>(a.group >> 3);
  for (int o = 1; o < lanes; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  float s = fmaxf(amax / 448.0f, 1.0f / (448.0f * 512.0f));
  const bool e8m0 = a.scale_dtype == MI355MOE_U8;
  int ex = 0;
  if (e8m0 || a.scale_ue8m0) {
    ex = ceil_log2(s);
    s = ex > 127 ? __uint_as_float(0x7F800000u) : pow2i(ex);  // an infinite maximum
  }
  const int64_t g = i / a.group;
  if (i % a.group == 0) {
    const int64_t at = r * a.scale_row + g * a.scale_group;
    if (e8m0) static_cast<uint8_t*>(a.scales)[at] = static_cast<uint8_t>(ex + 127);
    else static_cast<float*>(a.scales)[at] = s;
  }
  const float inv = 1.0f / s;
  const uint32_t lo = e4m3x4_nan(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
  const uint32_t hi = e4m3x4_nan(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
  uint8_t* q = static_cast<uint8_t*>(a.q) + r * a.cols + i;
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = static_cast<uint8_t>((k < 4 ? lo : hi) >> (8 * (k & 3)));
  }
}

template <typename E, bool VEC>
__global__ __launch_bounds__(256) void rms_norm_kernel(const NormArgs a) {
  const int64_t r = blockIdx.x;
  const char* x = static_cast<const char*>(a.x) + row_at<E>(r, a.inner, a.x_outer, a.x_inner);
  const char* res = a.residual ? static_cast<const char*>(a.residual) +
                                     row_at<E>(r, a.inner, a.residual_outer, a.residual_inner)
                               : nullptr;
  auto load_h = [&](int64_t i, float (&h)[8]) {
    load8<E, VEC>(x, i, a.cols, h);
    if (res) {
      float t[8];
      load8<E, VEC>(res, i, a.cols, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] += t[k];
    }
  };
  float ss = 0.f;
  for (int64_t i = threadIdx.x * 8; i < a.cols; i += 256 * 8) {
    float h[8];
    load_h(i, h);
#pragma unroll
    for (int k = 0; k < 8; ++k) ss += h[k] * h[k];
  }
  __shared__ float part[4];
  ss = wave_sum(ss);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  ss = (part[0] + part[1]) + (part[2] + part[3]);
  const float rs = 1.0f / sqrtf(ss / static_cast<float>(a.cols) + a.eps);
  for (int64_t i = threadIdx.x * 8; i < a.cols; i += 256 * 8) {
    float h[8], w[8], y[8];
    load_h(i, h);
    if (a.residual_out)
      store8<E, VEC>(static_cast<char*>(a.residual_out) +
                         row_at<E>(r, a.inner, a.residual_out_outer, a.residual_out_inner),
                     i, a.cols, h);
    if (a.weight_dtype == MI355MOE_F32) load8<F32, VEC>(a.weight, i, a.cols, w);
    else load8<E, VEC>(a.weight, i, a.cols, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = h[k] * rs * w[k];
    if (a.out)
      store8<E, VEC>(static_cast<char*>(a.out) + row_at<E>(r, a.inner, a.out_outer, a.out_inner),
                     i, a.cols, y);
    if (a.q) quant8<VEC>(a, r, i, y);
  }
}

bool mul16(const void* p, int64_t outer, int64_t inner, int64_t n_inner, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (outer * size) % 16 == 0 &&
         (n_inner == 1 || (inner * size) % 16 == 0);
}

template <typename E>
int launch(const NormArgs& a, hipStream_t st) {
  const int size = sizeof(typename E::T);
  const bool vec =
      a.cols % 8 == 0 && mul16(a.x, a.x_outer, a.x_inner, a.inner, size) &&
      (!a.residual ||
       (mul16(a.residual, a.residual_outer, a.residual_inner, a.inner, size) &&
        mul16(a.residual_out, a.residual_out_outer, a.residual_out_inner, a.inner, size))) &&
      (!a.out || mul16(a.out, a.out_outer, a.out_inner, a.inner, size)) &&
      mul16(a.weight, 0, 0, 1, 2) && (!a.q || (reinterpret_cast<uintptr_t>(a.q) & 7) == 0);
  const dim3 grid(static_cast<unsigned>(a.rows));
  if (vec) rms_norm_kernel<E, true><<<grid, dim3(256), 0, st>>>(a);
  else rms_norm_kernel<E, false><<<grid, dim3(256), 0, st>>>(a);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355moe_rms_norm(const mi355moe_rms_norm_args* p, void* stream) {
  MI_ARG(p, "null pointer");
  const NormArgs a = *p;
  MI_ARG(a.dtype == MI355MOE_F32 || a.dtype == MI355MOE_BF16 || a.dtype == MI355MOE_F16,
         "rms_norm: input must be float32, bfloat16 or float16");
  MI_ARG(a.weight_dtype == a.dtype || a.weight_dtype == MI355MOE_F32,
         "rms_norm: weight must have the input's type or be float32");
  MI_ARG(a.rows >= 0 && a.cols > 0 && a.inner > 0, "rms_norm: invalid shape");
  MI_ARG(a.rows <= 0x7FFFFFFF, "rms_norm: too many rows");
  MI_ARG((a.residual != nullptr) == (a.residual_out != nullptr) || a.rows == 0,
         "rms_norm: residual and residual_out go together");
  MI_ARG(a.out || a.q || a.rows == 0, "rms_norm: no output");
  if (a.q) {
    MI_ARG(a.group == 32 || a.group == 64 || a.group == 128,
           "rms_norm: group_size must be 32, 64 or 128");
    MI_ARG(a.cols % a.group == 0, "rms_norm: hidden size must be divisible by group_size");
    MI_ARG(a.scale_dtype == MI355MOE_F32 || a.scale_dtype == MI355MOE_U8,
           "rms_norm: scales must be float32 or e8m0 codes");
    MI_ARG(a.scales, "rms_norm: scales missing");
  }
  if (a.rows == 0) return MI355MOE_OK;
  MI_ARG(a.x && a.weight, "null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (a.dtype) {
    case MI355MOE_F32: return launch<F32>(a, st);
    case MI355MOE_BF16: return launch<BF16>(a, st);
    default: return launch<F16>(a, st);
  }
}
