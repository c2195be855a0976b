// Entry of mi355moe_linear (linear.h has the formulas) and its kernel for any
// size, stride and alignment: 64 x 64 output tiles (gated: 64 x 64 of both
// halves), 4 waves of 16 columns each, both operands' K stages copied through
// registers into LDS with zeros past the edges, so every K is exact.
#include "linear.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int GM = 64, GN = 64;

// K stages [split * per, ...) of 128 bytes; the next stage's rows are in registers
// while this one's products run.
// KEEP: the sums go to a.z too.  RAW (int8): a split's sums, as they are.
template <int KIND, bool GATED, bool KEEP, bool RAW>
__global__ __launch_bounds__(256) void linear_any_kernel(const LinArgs a, int per) {
  constexpr bool FP8 = KIND == K_FP8;
  using Sum = typename SumVec<KIND, 4>::T;
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
  constexpr int EB = kind_bytes(KIND);
  const int64_t kbytes = a.K * EB;
  const uint8_t* x = static_cast<const uint8_t*>(a.x);
  const uint8_t* w = static_cast<const uint8_t*>(a.weight);
  const int64_t kfirst = static_cast<int64_t>(blockIdx.z) * per * SB;
  const int64_t kend = kfirst + static_cast<int64_t>(per) * SB < kbytes
                           ? kfirst + static_cast<int64_t>(per) * SB : kbytes;

  Sum acc[NH][4];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[h][j] = Sum{0, 0, 0, 0};

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
            acc[h][j] = mfma_16x16<KIND>(av, bv, acc[h][j]);
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
      if constexpr (RAW) {
        static_cast<int*>(a.out)[part + m * a.ldo + n] = acc[0][j][r];
      } else if constexpr (KIND == K_I8) {
        st_any(a.out, a.out_dtype, part + m * a.ldo + n,
               lin_value_i32(a, m, n, x_scale_of(a, m), acc[0][j][r], acc[NH - 1][j][r]));
      } else {
        st_any(a.out, a.out_dtype, part + m * a.ldo + n,
               lin_value<KEEP>(a, m, n, acc[0][j][r], acc[NH - 1][j][r]));
      }
    }
  }
}

template <int KIND>
int launch_any(const LinArgs& a, int splits, int per, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, GN)), static_cast<unsigned>(cdiv(a.M, GM)),
                  static_cast<unsigned>(splits));
  constexpr bool W16 = KIND == K_BF16 || KIND == K_F16, I8 = KIND == K_I8;
  if (W16 && a.z) linear_any_kernel<KIND, true, W16, false><<<grid, dim3(256), 0, st>>>(a, per);
  else if (I8 && splits > 1) linear_any_kernel<KIND, false, false, I8><<<grid, dim3(256), 0, st>>>(a, per);
  else if (lin_gated(a.activation))
    linear_any_kernel<KIND, true, false, false><<<grid, dim3(256), 0, st>>>(a, per);
  else linear_any_kernel<KIND, false, false, false><<<grid, dim3(256), 0, st>>>(a, per);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

// K is split until there are about 1000 workgroups (four per CU), 8 stages each
// at least.
int any_stages(const LinArgs& a) {
  const int64_t nk = cdiv(a.K * kind_bytes(kind_of(a)), 128);
  const int64_t tiles = cdiv(a.M, GM) * cdiv(lin_rows(a), GN);
  const int64_t most = nk / 8 > 1 ? nk / 8 : 1, want = cdiv(1000, tiles);
  return static_cast<int>(cdiv(nk, want < most ? want : most));
}
int any_splits(const LinArgs& a) {
  return static_cast<int>(cdiv(cdiv(a.K * kind_bytes(kind_of(a)), 128), any_stages(a)));
}

// Split K: the sum of the splits' partial sums, in their order, then the epilogue.
// The loads of kAhead splits are on their way at once, and workgroups are one wave
// so that few outputs reach many CUs (24 x 4096 x 4096, both kernels: 13.9 us; one
// split after the other 15.3, four at once 14.5, workgroups of 256 14.0).
// I8: int32 partial sums.  KEEP: the sums go to a.z too.
template <bool GATED, bool I8, bool KEEP>
__global__ __launch_bounds__(64) void linear_finish_kernel(const LinArgs a,
                                                            const void* __restrict__ parts,
                                                            int splits, int64_t rows) {
  constexpr int kAhead = 8, H = GATED ? 2 : 1;
  using S = std::conditional_t<I8, int, float>;
  typedef typename SumVec<I8 ? K_I8 : K_BF16, 4>::T S4 __attribute__((aligned(4)));
  const S* part = static_cast<const S*>(parts);
  const int64_t chunks = (a.N + 7) / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  if (idx >= a.M * chunks) return;
  const int64_t m = idx / chunks, n = (idx % chunks) * 8;
  S z[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int k = 0; k < 8; ++k) z[h][k] = 0;
  const int64_t step = a.M * rows;
  const S* p = part + m * rows + n;
  if (n + 8 <= a.N) {
    for (int s = 0; s < splits; s += kAhead) {
      S4 v[kAhead][H][2];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const S* q = p + (s + e < splits ? s + e : splits - 1) * step;  // surplus: unused
#pragma unroll
        for (int h = 0; h < H; ++h) {
          v[e][h][0] = reinterpret_cast<const S4*>(q + h * a.N)[0];
          v[e][h][1] = reinterpret_cast<const S4*>(q + h * a.N)[1];
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
  const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * osize)) & 15) == 0;
  if constexpr (I8) lin_store8_i32(a, m, n, z[0], z[H - 1], vec);
  else lin_store8<KEEP>(a, m, n, z[0], z[H - 1], vec);
}

// 16-bit x that becomes int8 in the call
bool quantises(const LinArgs& a) {
  return a.weight_dtype == MI355MOE_I8 && a.x_dtype != MI355MOE_I8;
}

bool float_dtype(int d) {
  return d == MI355MOE_F32 || d == MI355MOE_BF16 || d == MI355MOE_F16;
}

int check(const LinArgs& a) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3, i8 = a.x_dtype == MI355MOE_I8;
  MI_ARG(fp8 || i8 || a.x_dtype == MI355MOE_BF16 || a.x_dtype == MI355MOE_F16,
         "linear: x must be bfloat16, float16 or float8_e4m3fn, or int8");
  MI_ARG(a.weight_dtype == 0 || a.weight_dtype == a.x_dtype || (a.weight_dtype == MI355MOE_I8 && !fp8),
         "linear: weight must have x's type, or be int8 for bfloat16 and float16 x");
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
  MI_ARG(!(i8 || quantises(a)) || a.K < (1 << 17), "linear: K must be below 131072 for int8 operands");
  MI_ARG(!a.z || (lin_gated(a.activation) && !fp8 && !i8 && !quantises(a)),
         "linear: z is kept for gated activations of 16-bit operands");
  MI_ARG(!a.z || (reinterpret_cast<uintptr_t>(a.z) & 15) == 0, "linear: z must be 16-byte aligned");
  MI_ARG(!a.z || (a.N <= (1 << 20) && a.K <= (1 << 24)), "linear: size too large for a backward pass");
  return MI355MOE_OK;
}

// Rows to multiples of 16 bytes, zeros behind them.
__global__ __launch_bounds__(256) void pack_rows_kernel(const uint8_t* __restrict__ src, int64_t ld,
                                                        int64_t bytes, uint8_t* __restrict__ dst,
                                                        int64_t pitch, int64_t rows) {
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 16;
  if (c >= pitch) return;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    *reinterpret_cast<uint4*>(dst + r * pitch + c) = row16(src + r * ld, true, c, bytes);
}

}  // namespace

int launch_pack_rows(const void* src, int64_t ld, int64_t bytes, void* dst, int64_t rows, hipStream_t st) {
  const int64_t pitch = (bytes + 15) / 16 * 16;
  const int64_t wide = cdiv(pitch, 4096);
  int64_t high = rows < 4096 ? rows : 4096;
  pack_rows_kernel<<<dim3(static_cast<unsigned>(wide), static_cast<unsigned>(high)), dim3(256), 0, st>>>(
      static_cast<const uint8_t*>(src), ld, bytes, static_cast<uint8_t*>(dst), pitch, rows);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

}  // namespace mi355

using namespace mi355;

namespace mi355 {
int launch_linear_finish(const LinArgs& a, const void* part, int splits, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.M * cdiv(a.N, 8), 64)));
  const int64_t rows = lin_rows(a);
  const bool i8 = a.x_dtype == MI355MOE_I8;
  if (lin_gated(a.activation)) {
    if (a.z) linear_finish_kernel<true, false, true><<<grid, dim3(64), 0, st>>>(a, part, splits, rows);
    else if (i8) linear_finish_kernel<true, true, false><<<grid, dim3(64), 0, st>>>(a, part, splits, rows);
    else linear_finish_kernel<true, false, false><<<grid, dim3(64), 0, st>>>(a, part, splits, rows);
  } else if (i8) {
    linear_finish_kernel<false, true, false><<<grid, dim3(64), 0, st>>>(a, part, splits, rows);
  } else {
    linear_finish_kernel<false, false, false><<<grid, dim3(64), 0, st>>>(a, part, splits, rows);
  }
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}
}  // namespace mi355

namespace {
size_t lin_partials(const LinArgs& a, int splits) {
  return splits == 1 ? 0 : static_cast<size_t>(splits) * a.M * lin_rows(a) * sizeof(float);
}
enum Path { SKINNY, TILE, ANY };
Path path_of(const LinArgs& a) {
  const bool tile = linear_tile_supported(a);
  if (!a.z && linear_skinny_takes(a, tile)) return SKINNY;
  return tile ? TILE : ANY;
}
int splits_of(const LinArgs& a, Path path) {
  return path == SKINNY ? 1 : path == TILE ? linear_tile_splits(a) : any_splits(a);
}
size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }
// How a call runs: on which operands, and what of them is made in the workspace before the
// partial sums.
struct Call {
  LinArgs a;          // the product that runs
  bool quant = false; // x becomes codes (rows at multiples of 16 bytes, zeros behind them) ...
  bool pack_x = false, pack_w = false;  // ... or is copied to such rows, as is the weight
  Path path = ANY;
  int splits = 1;
  size_t scales = 0, weight = 0, parts = 0, total = 0;  // offsets, and the whole
};
// Operands of int8 and of kept sums that direct copies cannot fetch are copied to rows that
// they can (launch_pack_rows), which pays where many rows share the copied weight (rows x K x
// weight rows, both kernels in us, through registers / copied: kept 1024 x 6709 x 4094 132 / 103,
// 512 x 1001 x 2002 27.6 / 22.3, 257 x 1001 x 1030 19.9 / 19.5, 100 x 6709 x 4094 44.8 / 50.2; int8
// gated 1024 x 6709 x 4094 89 / 63, 257 x 1001 x 1030 27.2 / 17.7, 100 x 6709 x 4094 38.2 / 40.0).
// Below 10^9 operations the launches of the copies cost a caller more than they save (a step of
// 257 x 1001 x 1030 from Python 68 / 78).
constexpr int64_t kPackRows = 256;
constexpr double kPackWork = 1e9;
Call call_of(const LinArgs& given, void* workspace) {
  Call c;
  c.a = given;
  LinArgs& a = c.a;
  const uintptr_t ws = reinterpret_cast<uintptr_t>(workspace);
  c.quant = quantises(given);
  if (c.quant && linear_skinny_quantises(given)) {
    c.path = SKINNY;  // by the kernel itself
    c.quant = false;
    return c;
  }
  size_t at = 0;
  if (c.quant) {
    a.ldx = static_cast<int64_t>(up16(static_cast<size_t>(a.K)));
    a.x_dtype = MI355MOE_I8;
    a.x = reinterpret_cast<const void*>(ws);
    c.scales = static_cast<size_t>(a.M) * a.ldx;
    a.x_scale = reinterpret_cast<const float*>(ws + c.scales);
    a.x_scale_row = 1;
    at = c.scales + up16(static_cast<size_t>(a.M) * sizeof(float));
  }
  c.path = path_of(a);
  if (c.path == ANY && (a.z || a.x_dtype == MI355MOE_I8) && a.M >= kPackRows &&
      2.0 * a.M * a.K * lin_rows(a) >= kPackWork) {
    const int64_t eb = kind_bytes(kind_of(a)), pitch = static_cast<int64_t>(up16(static_cast<size_t>(a.K * eb)));
    auto rows16 = [&](const void* p, int64_t ld) {
      return a.K * eb % 16 == 0 && ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * eb)) & 15) == 0;
    };
    LinArgs b = a;
    size_t end = at;
    c.pack_x = !c.quant && !rows16(a.x, a.ldx);
    if (c.pack_x) {
      b.x = reinterpret_cast<const void*>(ws + end);
      b.ldx = pitch / eb;
      end += static_cast<size_t>(a.M) * pitch;
    }
    c.pack_w = !rows16(a.weight, a.ldw);
    if (c.pack_w) {
      c.weight = end;
      b.weight = reinterpret_cast<const void*>(ws + end);
      b.ldw = pitch / eb;
      end += static_cast<size_t>(lin_rows(a)) * pitch;
    }
    b.K = pitch / eb;
    if (linear_tile_supported(b)) {
      a = b;
      at = end;
      c.path = TILE;
    } else {
      c.pack_x = c.pack_w = false;
    }
  }
  c.splits = splits_of(a, c.path);
  c.parts = at;
  c.total = at + lin_partials(a, c.splits);
  return c;
}
}  // namespace

extern "C" size_t mi355moe_linear_workspace_size(const mi355moe_linear_args* p) {
  if (!p || check(*p) || p->M == 0) return 0;
  return call_of(*p, nullptr).total;
}

extern "C" int mi355moe_linear(const mi355moe_linear_args* p, void* workspace,
                               size_t workspace_bytes, void* stream) {
  MI_ARG(p, "null pointer");
  const LinArgs given = *p;
  if (const int rc = check(given)) return rc;
  if (given.M == 0) return MI355MOE_OK;
  MI_ARG(given.x && given.weight && given.out, "null pointer");
  const bool i8 = given.x_dtype == MI355MOE_I8 || quantises(given);
  MI_ARG((given.x_dtype != MI355MOE_FP8E4M3 && !i8) ||
             ((given.x_scale || quantises(given)) && given.weight_scale), "linear: scales missing");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Call c = call_of(given, workspace);
  const LinArgs& a = c.a;
  MI_CHECK(c.total == 0 || (workspace && workspace_bytes >= c.total), MI355MOE_ERR_WORKSPACE,
           "linear: workspace too small");
  MI_ARG(c.total == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
         "linear: workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t eb = kind_bytes(kind_of(a));
  int rc = 0;
  if (c.quant)
    rc = launch_int8_quant(given.x_dtype, given.x, given.ldx, reinterpret_cast<int8_t*>(ws), a.ldx,
                           reinterpret_cast<float*>(ws + c.scales), 1, a.M, given.K, st, true);
  if (!rc && c.pack_x) rc = launch_pack_rows(given.x, given.ldx * eb, given.K * eb, ws, a.M, st);
  if (!rc && c.pack_w)
    rc = launch_pack_rows(given.weight, given.ldw * eb, given.K * eb, ws + c.weight, lin_rows(a), st);
  if (rc) return rc;
  if (c.path == SKINNY) return launch_linear_skinny(a, st);
  // a split product leaves partial sums (fp32, of int8 products int32) of all weight rows
  void* parts = ws + c.parts;
  LinArgs b = a;
  if (c.splits > 1) {
    b.N = b.ldo = lin_rows(a);
    b.activation = MI355MOE_LINEAR_NONE;
    b.bias = b.residual = nullptr;
    b.out = parts;
    b.out_dtype = MI355MOE_F32;
    b.z = nullptr;
  }
  if (c.path == TILE) {
    rc = launch_linear_tile(a, b, st);
  } else {
    const int per = any_stages(a);
    switch (kind_of(a)) {
      case K_FP8: rc = launch_any<K_FP8>(b, c.splits, per, st); break;
      case K_I8: rc = launch_any<K_I8>(b, c.splits, per, st); break;
      case K_F16: rc = launch_any<K_F16>(b, c.splits, per, st); break;
      default: rc = launch_any<K_BF16>(b, c.splits, per, st);
    }
  }
  if (rc || c.splits == 1) return rc;
  return launch_linear_finish(a, parts, c.splits, st);
}
