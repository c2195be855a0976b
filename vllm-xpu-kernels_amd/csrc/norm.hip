// Root-mean-square norm of rows with the residual's addition before it and its
// result in the input's type, in e4m3 with a scale per group of columns, or
// both (mi355moe_rms_norm).  Per row, in fp32:
//   h = x + residual,  y = h / sqrt(sum(h^2) / cols + eps) * weight
// and per group of columns of y the scale and codes of the group quantisers
// (per_token_group_fp8_quant's arithmetic; e8m0 scales as the mxfp8 layer's).
//
// Bound by HBM (each input read once, each output written once) from a few
// hundred rows on, by latency below.  A row stays in registers between the sum
// of its squares and the outputs: R chunks of 8 columns per lane, the row's
// lanes in one wave (rows up to 512 columns, several rows per wave) or in one
// workgroup.  Rows beyond the registers of 1024 lanes are read twice.
#include "common.h"

namespace mi355 {
namespace {

typedef mi355moe_rms_norm_args NormArgs;

// Elements i, i + step, .. i + 7 step of a row: two or one 16-byte loads when VEC
// (step 1, i a multiple of 8), else those below `cols` one by one and zeros.
template <typename E, bool VEC>
__device__ __forceinline__ void load8(const void* p, int64_t i, int64_t cols, float (&f)[8],
                                      int step = 1) {
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
    for (int k = 0; k < 8; ++k) f[k] = i + k * step < cols ? E::ld(q[k * step]) : 0.f;
  }
}
// 16 bytes; `nt`: past the caches (launch_rows has the rule)
typedef uint32_t norm_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t norm_u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put16(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                      bool nt) {
  const norm_u32x4 v = {a, b, c, d};
  if (nt) __builtin_nontemporal_store(v, static_cast<norm_u32x4*>(p));
  else *static_cast<norm_u32x4*>(p) = v;
}
template <typename E, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t i, int64_t cols, const float (&f)[8],
                                       bool nt, int step = 1) {
  typename E::T* q = static_cast<typename E::T*>(p) + i;
  if constexpr (VEC && sizeof(typename E::T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = static_cast<uint32_t>(E::st(f[2 * k])) |
             (static_cast<uint32_t>(E::st(f[2 * k + 1])) << 16);
    put16(q, w[0], w[1], w[2], w[3], nt);
  } else if constexpr (VEC) {
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(f[k]);
    put16(q, w[0], w[1], w[2], w[3], nt);
    put16(q + 4, w[4], w[5], w[6], w[7], nt);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k * step < cols) q[k * step] = E::st(f[k]);
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

__device__ __forceinline__ bool pow2_scales(const NormArgs& a) {
  return a.scale_dtype == MI355MOE_U8 || a.scale_ue8m0;
}

// The group's scale and the lane's 8 codes of columns i .. i + 7.  A group is
// G / 8 consecutive, aligned lanes; every lane of the wave takes part, those
// without columns (`active` false) with zeros.
// Power-of-two scales double where the maximum passes 448 2^e: a maximum within
// 2^-20 of that (fp32's error is below) is compared in 64 bits, as squares and
// without a root or division:  |h w| / sqrt(ss / cols + eps) <= 448 2^e  where
// (h w)^2 cols <= (448 2^e)^2 (ss + eps cols).  The sides are off by a few 2^-53
// each; 2^-39 of slack (2^-40 of the maximum, which the clamp takes off its
// code) leaves a maximum that the formula puts on the border below it.
template <bool VEC>
__device__ __forceinline__ void quant8(const NormArgs& a, int64_t r, int i, bool active,
                                       const float (&y)[8], const float (&h)[8],
                                       const float (&w)[8], double ss, bool nt) {
  float amax = 1e-10f;
#pragma unroll
  for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(y[k]));
  const int group = static_cast<int>(a.group);
  if (group == 128) {
    amax = row16_max(amax);
  } else {
    amax = fmaxf(amax, __shfl_xor(amax, 1, 64));
    amax = fmaxf(amax, __shfl_xor(amax, 2, 64));
    if (group == 64) amax = fmaxf(amax, __shfl_xor(amax, 4, 64));
  }
  if (!active) return;
  float s = fmaxf(amax / 448.0f, 1.0f / (448.0f * 512.0f));
  const bool e8m0 = a.scale_dtype == MI355MOE_U8;
  int ex = 0;
  if (pow2_scales(a)) {
    ex = ceil_log2(s);
    const int low = ceil_log2(s * (1.0f - 0x1p-20f)), high = ceil_log2(s * (1.0f + 0x1p-20f));
    if (low != high) {  // the same in all lanes of a group
      double m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmax(m, fabs(static_cast<double>(h[k]) * w[k]));
      for (int o = 1; o < (group >> 3); o <<= 1) m = fmax(m, __shfl_xor(m, o, 64));
      const double n = static_cast<double>(a.cols), t = ldexp(448.0, low);
      ex = m * m * n <= t * t * (1.0 + 0x1p-39) * (ss + a.eps * n) ? low : high;
    }
    s = ex > 127 ? __uint_as_float(0x7F800000u) : pow2i(ex);  // an infinite maximum
  }
  if ((i & (group - 1)) == 0) {
    const int64_t at = r * a.scale_row + (i / group) * a.scale_group;
    if (e8m0) static_cast<uint8_t*>(a.scales)[at] = static_cast<uint8_t>(ex + 127);
    else static_cast<float*>(a.scales)[at] = s;
  }
  const float inv = 1.0f / s;
  const uint32_t lo = e4m3x4_nan(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
  const uint32_t hi = e4m3x4_nan(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
  uint8_t* q = static_cast<uint8_t*>(a.q) + r * a.cols + i;
  if constexpr (VEC) {
    const norm_u32x2 v = {lo, hi};
    if (nt) __builtin_nontemporal_store(v, reinterpret_cast<norm_u32x2*>(q));
    else *reinterpret_cast<norm_u32x2*>(q) = v;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = static_cast<uint8_t>((k < 4 ? lo : hi) >> (8 * (k & 3)));
  }
}

// The row's sum of squares in T, in every lane of the row.
template <typename T>
__device__ __forceinline__ T wave_sum_of(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <typename T>
__device__ __forceinline__ T workgroup_sum(T v, int waves) {
  __shared__ T part[16];
  v = wave_sum_of(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  T s = 0;
  for (int w = 0; w < waves; ++w) s += part[w];
  return s;
}
template <typename T, int LANES, int R>
__device__ __forceinline__ T row_sum(const float (&h)[R][8], int lanes) {
  T ss = 0;
#pragma unroll
  for (int c = 0; c < R; ++c)
#pragma unroll
    for (int k = 0; k < 8; ++k) ss += static_cast<T>(h[c][k]) * h[c][k];
  if constexpr (LANES != 0) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    return ss;
  } else {
    return workgroup_sum(ss, lanes >> 6);
  }
}

// 1 / sqrt(ss / cols + eps): fp32's values with one Newton step each in 64 bits
// before the rounding (the 64-bit division and root take 0.5 us of a small call)
__device__ __forceinline__ float rsqrt_mean(double ss, int cols, float eps) {
  const double r0 = 1.0f / static_cast<float>(cols);  // cols < 2^24 is exact, above off by 2^-24
  const double inv = r0 * (2.0 - static_cast<double>(cols) * r0);
  const double v = ss * inv + eps;
  const float s0 = 1.0f / sqrtf(static_cast<float>(v));
  // zero, infinite and NaN roots, and those whose square leaves fp32, stand
  if (!(v > 1e-30 && v < 1e30)) return s0;
  const double s = s0;
  return static_cast<float>(s * (1.5 - 0.5 * v * s * s));
}

// LANES: lanes of a row inside a wave (8 to 64, 256 / LANES rows to a
// workgroup of 256), or 0: the workgroup's blockDim.x lanes are one row's.
template <typename E, bool VEC, int LANES, int R, bool QUANT>
__global__ __launch_bounds__(LANES ? 256 : 1024) void rms_norm_kernel(const NormArgs a, int64_t row0, bool nt) {
  const int lanes = LANES ? LANES : static_cast<int>(blockDim.x);
  const int t = LANES ? threadIdx.x % LANES : threadIdx.x;
  const int64_t r = row0 + (LANES ? static_cast<int64_t>(blockIdx.x) * (256 / LANES) +
                                       threadIdx.x / LANES
                                 : static_cast<int64_t>(blockIdx.x));
  const int cols = static_cast<int>(a.cols);
  const bool row = r < a.rows;
  const int64_t rr = row ? r : 0;
  const char* x = static_cast<const char*>(a.x) + row_at<E>(rr, a.inner, a.x_outer, a.x_inner);
  const char* res = a.residual ? static_cast<const char*>(a.residual) +
                                     row_at<E>(rr, a.inner, a.residual_outer, a.residual_inner)
                               : nullptr;
  // Chunk c of this lane: 8 consecutive columns; where rows start anywhere and
  // no group binds columns to lanes, 8 columns `lanes` apart, so that a wave's
  // accesses are runs of 64 columns (8192 x 7167 bf16 314 -> 268 us).
  const int step = VEC || QUANT ? 1 : lanes;
  const auto at = [&](int c) { return step == 1 ? (c * lanes + t) * 8 : c * lanes * 8 + t; };
  float h[R][8], w[R][8];
  bool on[R];
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const int i = at(c);
    on[c] = row && i < cols;
#pragma unroll
    for (int k = 0; k < 8; ++k) h[c][k] = 0.f;
    if (on[c]) load8<E, VEC>(x, i, cols, h[c], step);
  }
  if (res) {
#pragma unroll
    for (int c = 0; c < R; ++c) {
      float u[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (on[c]) load8<E, VEC>(res, at(c), cols, u, step);
#pragma unroll
      for (int k = 0; k < 8; ++k) h[c][k] += u[k];
    }
  }
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const int i = at(c);
#pragma unroll
    for (int k = 0; k < 8; ++k) w[c][k] = 0.f;
    if (on[c]) {
      if (a.weight_dtype == MI355MOE_F32) load8<F32, VEC>(a.weight, i, cols, w[c], step);
      else load8<E, VEC>(a.weight, i, cols, w[c], step);
    }
  }
  float rs;
  double ss = 0;  // where a border needs it
  if (QUANT && pow2_scales(a)) {  // uniform
    ss = row_sum<double, LANES, R>(h, lanes);
    rs = rsqrt_mean(ss, cols, a.eps);
  } else {
    rs = 1.0f / sqrtf(row_sum<float, LANES, R>(h, lanes) / static_cast<float>(cols) + a.eps);
  }
  char* res_out = a.residual_out ? static_cast<char*>(a.residual_out) +
                                       row_at<E>(rr, a.inner, a.residual_out_outer,
                                                 a.residual_out_inner)
                                 : nullptr;
  char* out = a.out ? static_cast<char*>(a.out) + row_at<E>(rr, a.inner, a.out_outer, a.out_inner)
                    : nullptr;
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const int i = at(c);
    if (res_out && on[c]) store8<E, VEC>(res_out, i, cols, h[c], nt, step);
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = h[c][k] * rs * w[c][k];
    if (out && on[c]) store8<E, VEC>(out, i, cols, y, nt, step);
    if constexpr (QUANT) quant8<VEC>(a, rr, i, on[c], y, h[c], w[c], ss, nt);
  }
}

// Rows of any length: the row is read again for the outputs (by the same
// lanes, so an output may be the input).
template <typename E, bool VEC>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(const NormArgs a, int64_t row0, bool nt) {
  const int64_t r = row0 + blockIdx.x;
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
  // (in 64 bits: rows this long leave fp32 sums of some hundred terms per lane)
  double ss = 0;
  for (int64_t i = threadIdx.x * 8; i < a.cols; i += 1024 * 8) {
    float h[8];
    load_h(i, h);
#pragma unroll
    for (int k = 0; k < 8; ++k) ss += static_cast<double>(h[k]) * h[k];
  }
  ss = workgroup_sum(ss, 16);
  const float rs = rsqrt_mean(ss, static_cast<int>(a.cols), a.eps);
  for (int64_t i0 = 0; i0 < a.cols; i0 += 1024 * 8) {  // uniform: groups exchange maxima
    const int64_t i = i0 + threadIdx.x * 8;
    const bool on = i < a.cols;
    float h[8] = {}, w[8] = {}, y[8];
    if (on) load_h(i, h);
    if (on && a.residual_out)
      store8<E, VEC>(static_cast<char*>(a.residual_out) +
                         row_at<E>(r, a.inner, a.residual_out_outer, a.residual_out_inner),
                     i, a.cols, h, nt);
    if (on) {
      if (a.weight_dtype == MI355MOE_F32) load8<F32, VEC>(a.weight, i, a.cols, w);
      else load8<E, VEC>(a.weight, i, a.cols, w);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = h[k] * rs * w[k];
    if (on && a.out)
      store8<E, VEC>(static_cast<char*>(a.out) + row_at<E>(r, a.inner, a.out_outer, a.out_inner),
                     i, a.cols, y, nt);
    if (a.q) quant8<VEC>(a, r, static_cast<int>(on ? i : 0), on, y, h, w, ss, nt);
  }
}

template <typename E, bool VEC, int LANES, int R>
void launch_one(const NormArgs& a, int64_t row0, int64_t rows, int threads, bool nt,
                hipStream_t st) {
  const int64_t per = LANES ? 256 / (LANES ? LANES : 1) : 1;
  const dim3 grid(static_cast<unsigned>(cdiv(rows, per)));
  if (a.q) rms_norm_kernel<E, VEC, LANES, R, true><<<grid, dim3(threads), 0, st>>>(a, row0, nt);
  else rms_norm_kernel<E, VEC, LANES, R, false><<<grid, dim3(threads), 0, st>>>(a, row0, nt);
}

template <typename E, bool VEC>
int launch_rows(const NormArgs& a, int64_t row0, int64_t rows, hipStream_t st) {
  const int64_t chunks = cdiv(a.cols, 8);
  // Outputs larger than the L2s of the 8 XCDs (32 MiB) cannot stay there for
  // their reader; stored past them they leave room for the rows still read
  // (8192 x 7168 with e4m3 107 -> 99 us, 2048 x 7168 34 -> 24).
  const int64_t size = sizeof(typename E::T);
  const bool nt = a.rows * a.cols *
                      ((a.out ? size : 0) + (a.residual ? size : 0) + (a.q ? 1 : 0)) >
                  (int64_t(32) << 20);
  if (chunks <= 8) launch_one<E, VEC, 8, 1>(a, row0, rows, 256, nt, st);
  else if (chunks <= 16) launch_one<E, VEC, 16, 1>(a, row0, rows, 256, nt, st);
  else if (chunks <= 32) launch_one<E, VEC, 32, 1>(a, row0, rows, 256, nt, st);
  else if (chunks <= 64) launch_one<E, VEC, 64, 1>(a, row0, rows, 256, nt, st);
  else {
    // One chunk per lane is the fastest wherever its many waves are few rounds
    // of the GPU or one workgroup's barrier is short (bf16 with a residual, 1 / 2 / 4
    // chunks: 1 x 7168 3.3 / 3.8 / 5.2 us, 512 x 7168 8.4 / 8.7 / 11.0, 8192 x
    // 4096 46.2 / 49.3 / 54.0); wide rows in numbers want two (1024 x 7168 15.3 /
    // 12.1 / 13.0, 8192 x 7168 96.1 / 91.4 / 104.9).
    const int r = chunks <= 512 || (chunks <= 1024 && a.rows < 768) ? 1 : chunks <= 2048 ? 2 : 4;
    const int threads = static_cast<int>(cdiv(cdiv(chunks, r), 64) * 64);
    if (threads > 1024)
      rms_norm_long_kernel<E, VEC><<<dim3(static_cast<unsigned>(rows)), dim3(1024), 0, st>>>(a, row0, nt);
    else if (r == 1) launch_one<E, VEC, 0, 1>(a, row0, rows, threads, nt, st);
    else if (r == 2) launch_one<E, VEC, 0, 2>(a, row0, rows, threads, nt, st);
    else launch_one<E, VEC, 0, 4>(a, row0, rows, threads, nt, st);
  }
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
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
  // a launch's threads stay below 2^32
  constexpr int64_t kRows = int64_t(1) << 21;
  for (int64_t row0 = 0; row0 < a.rows; row0 += kRows) {
    const int64_t rows = a.rows - row0 < kRows ? a.rows - row0 : kRows;
    const int rc = vec ? launch_rows<E, true>(a, row0, rows, st)
                       : launch_rows<E, false>(a, row0, rows, st);
    if (rc) return rc;
  }
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
  MI_ARG(a.cols <= (1 << 28), "rms_norm: size too large");
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
