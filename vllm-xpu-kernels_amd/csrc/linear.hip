// Entry of mi355moe_linear (linear.h has the formulas) and its kernel for any
// size, stride and alignment: 64 x 64 output tiles (gated: 64 x 64 of both
// halves), 4 waves of 16 columns each, both operands' K stages copied through
// registers into LDS with zeros past the edges, so every K is exact.
#include "linear.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int GM = 64, GN = 64;

// 16 bytes from column byte c of a row of `bytes` bytes; zeros past its end
// and for rows that do not exist.
template <bool VEC>
__device__ __forceinline__ uint4 row16(const uint8_t* row, bool ok, int64_t c, int64_t bytes) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (!ok || c >= bytes) return v;
  if constexpr (VEC) {
    v = *reinterpret_cast<const uint4*>(row + c);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (c + k < bytes) w[k >> 2] |= static_cast<uint32_t>(row[c + k]) << (8 * (k & 3));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// VEC: rows of x and weight start at multiples of 16 bytes and are whole
// multiples of 16 bytes long.
template <bool FP8, bool F16, bool GATED, bool VEC>
__global__ __launch_bounds__(256) void linear_any_kernel(const LinArgs a) {
  constexpr int SB = FP8 ? 128 : 64;     // bytes of a K stage per row (128 e4m3 / 32 16-bit)
  constexpr int PITCH = SB + 16;
  constexpr int WR = GATED ? 2 * GN : GN;
  constexpr int NH = GATED ? 2 : 1;
  __shared__ __attribute__((aligned(16))) uint8_t sx[GM * PITCH];
  __shared__ __attribute__((aligned(16))) uint8_t sw[WR * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, q = lane >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * GM;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * GN;
  constexpr int EB = FP8 ? 1 : 2;
  const int64_t kbytes = a.K * EB;
  const uint8_t* x = static_cast<const uint8_t*>(a.x);
  const uint8_t* w = static_cast<const uint8_t*>(a.weight);

  f32x4 acc[NH][4];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int64_t k0 = 0; k0 < kbytes; k0 += SB) {
    __syncthreads();  // the previous stage is read
    for (int i = tid; i < GM * (SB / 16); i += 256) {
      const int r = i / (SB / 16), c = (i % (SB / 16)) * 16;
      const int64_t m = m0 + r;
      *reinterpret_cast<uint4*>(sx + r * PITCH + c) =
          row16<VEC>(x + m * a.ldx * EB, m < a.M, k0 + c, kbytes);
    }
    for (int i = tid; i < WR * (SB / 16); i += 256) {
      const int r = i / (SB / 16), c = (i % (SB / 16)) * 16;
      const int64_t n = n0 + (GATED ? r % GN : r);
      const int64_t row = n + (GATED && r >= GN ? a.N : 0);
      *reinterpret_cast<uint4*>(sw + r * PITCH + c) =
          row16<VEC>(w + row * a.ldw * EB, n < a.N, k0 + c, kbytes);
    }
    __syncthreads();
    if constexpr (FP8) {
      const int64_t kb = k0 / 128;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        // e4m3 to bf16 is exact, so the block's sum has fp32's precision (the
        // 128-long e4m3 product's has not, see linear.h)
        uint4 av[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          av[t] = fp8x8_to16<false, false>(*reinterpret_cast<const uint2*>(
              sw + (h * GN + 16 * wave + l16) * PITCH + 32 * t + 8 * q));
        // scales of the lane's 4 weight rows (row blocks of 128 over all rows)
        float ws[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t n = n0 + 16 * wave + 4 * q + r;
          ws[r] = n < a.N ? a.weight_scale[((n + (h ? a.N : 0)) / 128) * a.weight_scale_row +
                                           kb * a.weight_scale_blk]
                          : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < 4; ++t)
            d = mfma16_16x16x32<false>(
                av[t], fp8x8_to16<false, false>(*reinterpret_cast<const uint2*>(
                           sx + (16 * j + l16) * PITCH + 32 * t + 8 * q)), d);
          const int64_t m = m0 + 16 * j + l16;
          const float xs = m < a.M ? a.x_scale[m * a.x_scale_row + kb * a.x_scale_blk] : 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[h][j][r] += d[r] * (xs * ws[r]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint4 av = *reinterpret_cast<const uint4*>(sw + (h * GN + 16 * wave + l16) * PITCH + 16 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 bv = *reinterpret_cast<const uint4*>(sx + (16 * j + l16) * PITCH + 16 * q);
          acc[h][j] = mfma16_16x16x32<F16>(av, bv, acc[h][j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t m = m0 + 16 * j + l16;
    if (m >= a.M) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t n = n0 + 16 * wave + 4 * q + r;
      if (n >= a.N) continue;
      st_any(a.out, a.out_dtype, m * a.ldo + n,
             lin_value(a, m, n, acc[0][j][r], acc[NH - 1][j][r]));
    }
  }
}

template <bool FP8, bool F16>
int launch_any(const LinArgs& a, bool vec, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, GN)), static_cast<unsigned>(cdiv(a.M, GM)));
  const bool g = lin_gated(a.activation);
  if (g && vec) linear_any_kernel<FP8, F16, true, true><<<grid, dim3(256), 0, st>>>(a);
  else if (g) linear_any_kernel<FP8, F16, true, false><<<grid, dim3(256), 0, st>>>(a);
  else if (vec) linear_any_kernel<FP8, F16, false, true><<<grid, dim3(256), 0, st>>>(a);
  else linear_any_kernel<FP8, F16, false, false><<<grid, dim3(256), 0, st>>>(a);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

bool float_dtype(int d) {
  return d == MI355MOE_F32 || d == MI355MOE_BF16 || d == MI355MOE_F16;
}

int check(const LinArgs& a) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  MI_ARG(fp8 || a.x_dtype == MI355MOE_BF16 || a.x_dtype == MI355MOE_F16,
         "linear: x must be bfloat16, float16 or float8_e4m3fn");
  MI_ARG(float_dtype(a.out_dtype), "linear: out must be float32, bfloat16 or float16");
  MI_ARG(!a.bias || float_dtype(a.bias_dtype), "linear: bias must be float32, bfloat16 or float16");
  MI_ARG(!a.residual || float_dtype(a.residual_dtype),
         "linear: residual must be float32, bfloat16 or float16");
  MI_ARG(a.activation >= MI355MOE_LINEAR_NONE && a.activation <= MI355MOE_LINEAR_GELU_TANH_AND_MUL,
         "linear: unknown activation");
  MI_ARG(a.M >= 0 && a.N > 0 && a.K > 0, "linear: invalid shape");
  MI_ARG(a.M <= 64 * 65535 && a.N <= (1 << 28) && a.K <= (1 << 28), "linear: size too large");
  MI_ARG(!fp8 || a.K % 128 == 0, "linear: K must be divisible by 128 for float8 operands");
  return MI355MOE_OK;
}

}  // namespace
}  // namespace mi355

using namespace mi355;

namespace {
enum Path { SKINNY, TILE, ANY };
Path path_of(const LinArgs& a) {
  if (linear_skinny_takes(a)) return SKINNY;
  return linear_tile_supported(a) ? TILE : ANY;
}
}  // namespace

extern "C" size_t mi355moe_linear_workspace_size(const mi355moe_linear_args* p) {
  if (!p || check(*p) || p->M == 0) return 0;
  return path_of(*p) == TILE ? linear_tile_workspace(*p) : 0;
}

extern "C" int mi355moe_linear(const mi355moe_linear_args* p, void* workspace,
                               size_t workspace_bytes, void* stream) {
  MI_ARG(p, "null pointer");
  const LinArgs a = *p;
  if (const int rc = check(a)) return rc;
  if (a.M == 0) return MI355MOE_OK;
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  MI_ARG(a.x && a.weight && a.out, "null pointer");
  MI_ARG(!fp8 || (a.x_scale && a.weight_scale), "linear: scales missing");
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (path_of(a)) {
    case SKINNY: return launch_linear_skinny(a, st);
    case TILE: {
      const size_t need = linear_tile_workspace(a);
      MI_CHECK(need == 0 || (workspace && workspace_bytes >= need), MI355MOE_ERR_WORKSPACE,
               "linear: workspace too small");
      return launch_linear_tile(a, workspace, st);
    }
    default: break;
  }
  const int eb = fp8 ? 1 : 2;
  auto rows16 = [&](const void* p_, int64_t ld) {
    return ((reinterpret_cast<uintptr_t>(p_) | static_cast<uintptr_t>(ld * eb)) & 15) == 0;
  };
  const bool vec = rows16(a.x, a.ldx) && rows16(a.weight, a.ldw) && a.K * eb % 16 == 0;
  if (fp8) return launch_any<true, false>(a, vec, st);
  return a.x_dtype == MI355MOE_F16 ? launch_any<false, true>(a, vec, st)
                                   : launch_any<false, false>(a, vec, st);
}
