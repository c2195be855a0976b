// Entry of mi355moe_linear (linear.h has the formulas) and its kernel for any
// size, stride and alignment: 64 x 64 output tiles (gated: 64 x 64 of both
// halves), 4 waves of 16 columns each, both operands' K stages copied through
// registers into LDS with zeros past the edges, so every K is exact.
#include "linear.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int GM = 64, GN = 64;

// 16 bytes from column byte c of a row of `bytes` bytes, from any address;
// zeros past its end and for rows that do not exist.
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

// K stages [split * per, ...) of 128 bytes; the next stage's rows are in registers
// while this one's products run.
template <bool FP8, bool F16, bool GATED>
__global__ __launch_bounds__(256) void linear_any_kernel(const LinArgs a, int per) {
  constexpr int SB = 128;                // bytes of a K stage per row
  constexpr int PITCH = SB + 16;
  constexpr int WR = GATED ? 2 * GN : GN;
  constexpr int NH = GATED ? 2 : 1;
  constexpr int XC = GM * (SB / 16) / 256, WC = WR * (SB / 16) / 256;  // 16-byte pieces per thread
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
  const int64_t kfirst = static_cast<int64_t>(blockIdx.z) * per * SB;
  const int64_t kend = kfirst + static_cast<int64_t>(per) * SB < kbytes
                           ? kfirst + static_cast<int64_t>(per) * SB : kbytes;

  f32x4 acc[NH][4];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[h][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  uint4 px[XC], pw[WC];
  auto fetch = [&](int64_t k) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < XC; ++e) {
      const int i = e * 256 + tid;
      const int64_t m = m0 + i / (SB / 16);
      px[e] = row16(x + m * a.ldx * EB, m < a.M, k + (i % (SB / 16)) * 16, kbytes);
    }
#pragma unroll
    for (int e = 0; e < WC; ++e) {
      const int i = e * 256 + tid, r = i / (SB / 16);
      const int64_t n = n0 + (GATED ? r % GN : r);
      pw[e] = row16(w + (n + (GATED && r >= GN ? a.N : 0)) * a.ldw * EB, n < a.N,
                    k + (i % (SB / 16)) * 16, kbytes);
    }
  };
  fetch(kfirst);
  for (int64_t k0 = kfirst; k0 < kend; k0 += SB) {
    __syncthreads();  // the previous stage is read
#pragma unroll
    for (int e = 0; e < XC; ++e) {
      const int i = e * 256 + tid;
      *reinterpret_cast<uint4*>(sx + (i / (SB / 16)) * PITCH + (i % (SB / 16)) * 16) = px[e];
    }
#pragma unroll
    for (int e = 0; e < WC; ++e) {
      const int i = e * 256 + tid;
      *reinterpret_cast<uint4*>(sw + (i / (SB / 16)) * PITCH + (i % (SB / 16)) * 16) = pw[e];
    }
    __syncthreads();
    if (k0 + SB < kend) fetch(k0 + SB);  // uniform
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
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const uint4 av = *reinterpret_cast<const uint4*>(sw + (h * GN + 16 * wave + l16) * PITCH +
                                                           64 * t + 16 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 bv = *reinterpret_cast<const uint4*>(sx + (16 * j + l16) * PITCH + 64 * t + 16 * q);
            acc[h][j] = mfma16_16x16x32<F16>(av, bv, acc[h][j]);
          }
        }
      }
    }
  }
  // a split writes its partial sums (float32 outputs without an epilogue)
  const int64_t part = static_cast<int64_t>(blockIdx.z) * a.M * a.ldo;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t m = m0 + 16 * j + l16;
    if (m >= a.M) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t n = n0 + 16 * wave + 4 * q + r;
      if (n >= a.N) continue;
      st_any(a.out, a.out_dtype, part + m * a.ldo + n,
             lin_value(a, m, n, acc[0][j][r], acc[NH - 1][j][r]));
    }
  }
}

template <bool FP8, bool F16>
int launch_any(const LinArgs& a, int splits, int per, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, GN)), static_cast<unsigned>(cdiv(a.M, GM)),
                  static_cast<unsigned>(splits));
  if (lin_gated(a.activation)) linear_any_kernel<FP8, F16, true><<<grid, dim3(256), 0, st>>>(a, per);
  else linear_any_kernel<FP8, F16, false><<<grid, dim3(256), 0, st>>>(a, per);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

// K is split until there are about 1000 workgroups (four per CU), 8 stages each
// at least.
int any_stages(const LinArgs& a) {
  const int64_t nk = cdiv(a.K * (a.x_dtype == MI355MOE_FP8E4M3 ? 1 : 2), 128);
  const int64_t tiles = cdiv(a.M, GM) * cdiv(lin_rows(a), GN);
  const int64_t most = nk / 8 > 1 ? nk / 8 : 1, want = cdiv(1000, tiles);
  return static_cast<int>(cdiv(nk, want < most ? want : most));
}
int any_splits(const LinArgs& a) {
  return static_cast<int>(cdiv(cdiv(a.K * (a.x_dtype == MI355MOE_FP8E4M3 ? 1 : 2), 128), any_stages(a)));
}

// Split K: the sum of the splits' partial sums, in their order, then the epilogue.
// The loads of kAhead splits are on their way at once, and workgroups are one wave
// so that few outputs reach many CUs (24 x 4096 x 4096, both kernels: 13.9 us; one
// split after the other 15.3, four at once 14.5, workgroups of 256 14.0).
template <bool GATED>
__global__ __launch_bounds__(64) void linear_finish_kernel(const LinArgs a,
                                                            const float* __restrict__ part,
                                                            int splits, int64_t rows) {
  constexpr int kAhead = 8, H = GATED ? 2 : 1;
  const int64_t chunks = (a.N + 7) / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  if (idx >= a.M * chunks) return;
  const int64_t m = idx / chunks, n = (idx % chunks) * 8;
  float z[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int k = 0; k < 8; ++k) z[h][k] = 0.f;
  const int64_t step = a.M * rows;
  const float* p = part + m * rows + n;
  if ((rows & 3) == 0 && (a.N & 3) == 0 && n + 8 <= a.N) {
    for (int s = 0; s < splits; s += kAhead) {
      f32x4 v[kAhead][H][2];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const float* q = p + (s + e < splits ? s + e : splits - 1) * step;  // surplus: unused
#pragma unroll
        for (int h = 0; h < H; ++h) {
          v[e][h][0] = reinterpret_cast<const f32x4*>(q + h * a.N)[0];
          v[e][h][1] = reinterpret_cast<const f32x4*>(q + h * a.N)[1];
        }
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (s + e < splits) {
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int k = 0; k < 8; ++k) z[h][k] += v[e][h][k >> 2][k & 3];
        }
    }
  } else {
    for (int s = 0; s < splits; ++s, p += step)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < a.N) {
          z[0][k] += p[k];
          if constexpr (GATED) z[1][k] += p[a.N + k];
        }
  }
  const int osize = a.out_dtype == MI355MOE_F32 ? 4 : 2;
  lin_store8(a, m, n, z[0], z[H - 1],
             ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * osize)) & 15) == 0);
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
  // grids and their threads are counted in 32 bits (4 weight rows to a workgroup)
  MI_ARG(a.M <= 64 * 65535 && a.N <= (1 << 24) && a.K <= (1 << 28), "linear: size too large");
  MI_ARG(a.ldx >= 0 && a.ldw >= 0 && a.ldr >= 0 && a.ldo >= 0 && a.x_scale_row >= 0 &&
             a.x_scale_blk >= 0 && a.weight_scale_row >= 0 && a.weight_scale_blk >= 0,
         "linear: negative stride");
  MI_ARG(a.M <= 1 || a.ldo >= a.N, "linear: rows of out overlap");
  MI_ARG(!fp8 || a.K % 128 == 0, "linear: K must be divisible by 128 for float8 operands");
  return MI355MOE_OK;
}

}  // namespace
}  // namespace mi355

using namespace mi355;

namespace {
int launch_linear_finish(const LinArgs& a, const float* part, int splits, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.M * cdiv(a.N, 8), 64)));
  if (lin_gated(a.activation))
    linear_finish_kernel<true><<<grid, dim3(64), 0, st>>>(a, part, splits, lin_rows(a));
  else linear_finish_kernel<false><<<grid, dim3(64), 0, st>>>(a, part, splits, lin_rows(a));
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}
size_t lin_partials(const LinArgs& a, int splits) {
  return splits == 1 ? 0 : static_cast<size_t>(splits) * a.M * lin_rows(a) * sizeof(float);
}
enum Path { SKINNY, TILE, ANY };
Path path_of(const LinArgs& a) {
  const bool tile = linear_tile_supported(a);
  if (linear_skinny_takes(a, tile)) return SKINNY;
  return tile ? TILE : ANY;
}
}  // namespace

extern "C" size_t mi355moe_linear_workspace_size(const mi355moe_linear_args* p) {
  if (!p || check(*p) || p->M == 0) return 0;
  const Path path = path_of(*p);
  return path == SKINNY ? 0
                        : lin_partials(*p, path == TILE ? linear_tile_splits(*p) : any_splits(*p));
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
  const Path path = path_of(a);
  if (path == SKINNY) return launch_linear_skinny(a, st);
  const int splits = path == TILE ? linear_tile_splits(a) : any_splits(a);
  MI_CHECK(splits == 1 || (workspace && workspace_bytes >= lin_partials(a, splits)),
           MI355MOE_ERR_WORKSPACE, "linear: workspace too small");
  MI_ARG(splits == 1 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
         "linear: workspace must be 16-byte aligned");
  // a split product leaves fp32 partial sums of all weight rows
  LinArgs b = a;
  if (splits > 1) {
    b.N = b.ldo = lin_rows(a);
    b.activation = MI355MOE_LINEAR_NONE;
    b.bias = b.residual = nullptr;
    b.out = workspace;
    b.out_dtype = MI355MOE_F32;
  }
  int rc;
  if (path == TILE) rc = launch_linear_tile(a, b, st);
  else if (fp8) rc = launch_any<true, false>(b, splits, any_stages(a), st);
  else if (a.x_dtype == MI355MOE_F16) rc = launch_any<false, true>(b, splits, any_stages(a), st);
  else rc = launch_any<false, false>(b, splits, any_stages(a), st);
  if (rc || splits == 1) return rc;
  return launch_linear_finish(a, static_cast<const float*>(workspace), splits, st);
}
