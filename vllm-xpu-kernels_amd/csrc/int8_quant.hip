// Rows to int8 codes with a scale each (mi355moe_int8_quant), per row in fp32:
//   s = max(max |x|, 1e-10) * fl(1 / 127),  q = rint(fl(x / s))
// each rounded to nearest, so that the codes are the formula's whatever computes them.
//
// Bound by HBM (each input read once, a byte written for it) from some hundred
// rows on, by latency below.  A row stays in registers between its maximum and its
// codes: R chunks of 8 columns per lane, the row's lanes in one wave (4 rows to a
// workgroup) or in one workgroup.  Longer rows are read twice.  16 x 4096 in fp16 2.6 us,
// 1003 x 2880 in bf16 4.8, 8192 x 7168 39 (4.5 TB/s; a large copy reaches 5.2).
#include "int8_quant.h"

namespace mi355 {
namespace {

struct QuantArgs {
  const void* x;
  int64_t ldx;
  int8_t* q;
  int64_t ldq;
  float* scales;
  int64_t scale_row, rows, cols;
  int pad;  // zeros behind a row's codes: below 16
};

__device__ __forceinline__ uint32_t workgroup_top(uint32_t m, int waves) {
  __shared__ uint32_t part[16];
  m = wave_top(m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = 0;
  for (int w = 0; w < waves; ++w) m = part[w] > m ? part[w] : m;
  return m;
}

template <bool VEC>
__device__ __forceinline__ void put8(int8_t* q, int64_t i, int64_t cols, uint2 w) {
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(q + i) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < cols) q[i + k] = static_cast<int8_t>((k < 4 ? w.x : w.y) >> (8 * (k & 3)));
  }
}

// WAVE: a row per wave, 4 to a workgroup; else a row per workgroup.
template <typename E, bool VEC, bool WAVE, int R>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void int8_quant_kernel(const QuantArgs a, int64_t row0) {
  const int lanes = WAVE ? 64 : static_cast<int>(blockDim.x);
  const int t = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int64_t r = row0 + (WAVE ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)
                                 : static_cast<int64_t>(blockIdx.x));
  if (WAVE && r >= a.rows) return;  // the wave's row
  const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
  float f[R][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const int64_t i = static_cast<int64_t>(c * lanes + t) * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) f[c][k] = 0.f;
    if (i < a.cols) row8<E, VEC>(x, i, a.cols, f[c]);
  }
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const uint32_t u = top8(f[c]);
    top = u > top ? u : top;
  }
  top = WAVE ? wave_top(top) : workgroup_top(top, lanes >> 6);
  const float s = scale_of(top);
  if (t == 0) a.scales[r * a.scale_row] = s;
  if (a.pad && t < a.pad) a.q[r * a.ldq + a.cols + t] = 0;
#pragma unroll
  for (int c = 0; c < R; ++c) {
    const int64_t i = static_cast<int64_t>(c * lanes + t) * 8;
    if (i < a.cols) put8<VEC>(a.q + r * a.ldq, i, a.cols, codes8(f[c], s));
  }
}

template <typename E, bool VEC>
__global__ __launch_bounds__(1024) void int8_quant_long_kernel(const QuantArgs a, int64_t row0) {
  const int64_t r = row0 + blockIdx.x;
  const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
  uint32_t top = 0;
  for (int64_t i = threadIdx.x * 8; i < a.cols; i += 1024 * 8) {
    float f[8];
    row8<E, VEC>(x, i, a.cols, f);
    const uint32_t u = top8(f);
    top = u > top ? u : top;
  }
  top = workgroup_top(top, 16);
  const float s = scale_of(top);
  if (threadIdx.x == 0) a.scales[r * a.scale_row] = s;
  if (threadIdx.x < a.pad) a.q[r * a.ldq + a.cols + threadIdx.x] = 0;
  for (int64_t i = threadIdx.x * 8; i < a.cols; i += 1024 * 8) {
    float f[8];
    row8<E, VEC>(x, i, a.cols, f);
    put8<VEC>(a.q + r * a.ldq, i, a.cols, codes8(f, s));
  }
}

template <typename E, bool VEC>
int launch_rows(const QuantArgs& a, int64_t row0, int64_t rows, hipStream_t st) {
  const int64_t chunks = cdiv(a.cols, 8);
  if (chunks <= 256) {
    const dim3 grid(static_cast<unsigned>(cdiv(rows, 4)));
    if (chunks <= 64) int8_quant_kernel<E, VEC, true, 1><<<grid, dim3(256), 0, st>>>(a, row0);
    else if (chunks <= 128) int8_quant_kernel<E, VEC, true, 2><<<grid, dim3(256), 0, st>>>(a, row0);
    else int8_quant_kernel<E, VEC, true, 4><<<grid, dim3(256), 0, st>>>(a, row0);
  } else {
    const dim3 grid(static_cast<unsigned>(rows));
    const int r = chunks <= 512 || (chunks <= 1024 && rows < 768) ? 1 : chunks <= 2048 ? 2 : 4;
    const int threads = static_cast<int>(cdiv(cdiv(chunks, r), 64) * 64);
    if (chunks > 4096) int8_quant_long_kernel<E, VEC><<<grid, dim3(1024), 0, st>>>(a, row0);
    else if (r == 1) int8_quant_kernel<E, VEC, false, 1><<<grid, dim3(threads), 0, st>>>(a, row0);
    else if (r == 2) int8_quant_kernel<E, VEC, false, 2><<<grid, dim3(threads), 0, st>>>(a, row0);
    else int8_quant_kernel<E, VEC, false, 4><<<grid, dim3(threads), 0, st>>>(a, row0);
  }
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

template <typename E>
int launch(const QuantArgs& a, hipStream_t st) {
  const bool vec = a.cols % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx * sizeof(typename E::T))) & 15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.ldq)) & 7) == 0;
  constexpr int64_t kRows = int64_t(1) << 21;  // a launch's threads stay below 2^32
  for (int64_t row0 = 0; row0 < a.rows; row0 += kRows) {
    const int64_t rows = a.rows - row0 < kRows ? a.rows - row0 : kRows;
    const int rc = vec ? launch_rows<E, true>(a, row0, rows, st) : launch_rows<E, false>(a, row0, rows, st);
    if (rc) return rc;
  }
  return MI355MOE_OK;
}

}  // namespace

int launch_int8_quant(int dtype, const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scales,
                      int64_t scale_row, int64_t rows, int64_t cols, hipStream_t st, bool pad) {
  const QuantArgs a{x, ldx, q, ldq, scales, scale_row, rows, cols,
                    pad ? static_cast<int>((16 - cols % 16) % 16) : 0};
  switch (dtype) {
    case MI355MOE_F32: return launch<F32>(a, st);
    case MI355MOE_BF16: return launch<BF16>(a, st);
    default: return launch<F16>(a, st);
  }
}

}  // namespace mi355

using namespace mi355;

extern "C" int mi355moe_int8_quant(const void* x, int dtype, int64_t ldx, int8_t* q, int64_t ldq,
                                   float* scales, int64_t scale_row, int64_t rows, int64_t cols,
                                   void* stream) {
  MI_ARG(dtype == MI355MOE_F32 || dtype == MI355MOE_BF16 || dtype == MI355MOE_F16,
         "int8_quant: input must be float32, bfloat16 or float16");
  MI_ARG(rows >= 0 && cols > 0, "int8_quant: invalid shape");
  MI_ARG(cols <= (1 << 28), "int8_quant: size too large");
  MI_ARG(ldx >= 0 && scale_row >= 0, "int8_quant: negative stride");
  MI_ARG(rows <= 1 || (ldq >= cols && scale_row >= 1), "int8_quant: rows of an output overlap");
  if (rows == 0) return MI355MOE_OK;
  MI_ARG(x && q && scales, "null pointer");
  return launch_int8_quant(dtype, x, ldx, q, ldq, scales, scale_row, rows, cols,
                           static_cast<hipStream_t>(stream));
}
