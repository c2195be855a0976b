// mi355moe_linear for few rows of x: a stream over the weight.
//
// A workgroup owns a strip of weight rows for all rows of x; its waves split
// K, each walks its range on its own (no LDS, no barrier), and the waves'
// sums meet in LDS in a fixed order.
//
// The 16 rows of the MFMA's A operand are R weight rows times C = 16 / R
// consecutive K chunks, its 16 columns R rows of x times the same C chunks: the
// product's blocks on the diagonal (row chunk = column chunk) hold the sums, the
// others are not used.  The matrix cores idle here anyway, while a strip of 4
// rows gives four times the workgroups that one of 16 does and reads each row
// in runs of 256 bytes instead of 64 (R = 4: up to 4 rows of x, 8: up to 8,
// 16: up to 16 per group of columns, MT groups).
//
// e4m3 operands are converted to bf16 (exact) as they arrive; each K step's
// product is multiplied by its blocks' scales, held in LDS.
#include "linear.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes from any address (gfx950 loads need no alignment)
typedef u32x4 __attribute__((aligned(1))) u32x4_any;
__device__ __forceinline__ u32x4 ld16_any(const uint8_t* p) {
  return *reinterpret_cast<const u32x4_any*>(p);
}
__device__ __forceinline__ uint4 as4(u32x4 v) { return make_uint4(v.x, v.y, v.z, v.w); }

constexpr int kScaleBytes = 48 * 1024;  // LDS for the e4m3 scales

template <bool FP8, bool F16, bool GATED, int R, int MT, int U>
__global__ __launch_bounds__(256) void linear_skinny_kernel(const LinArgs a) {
  constexpr int C = 16 / R;
  constexpr int STEP = C * 64;                // bytes of a row per K step
  constexpr int NS = GATED ? 2 : 1;           // strips: the gate's, the factor's
  constexpr int EB = FP8 ? 1 : 2;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = static_cast<int>(blockDim.x) >> 6;
  const int l16 = lane & 15, q = lane >> 4;
  const int ri = l16 % R, ci = l16 / R;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * R;
  const int64_t mbase = static_cast<int64_t>(blockIdx.y) * (R * MT);
  const int kbytes = static_cast<int>(a.K) * EB, kfull = kbytes & ~15;  // K <= 2^28

  // row n0 + ri of each strip; rows past the edges repeat the last one and are
  // not stored
  const uint8_t* wp[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    int64_t n = n0 + ri;
    n = (n < a.N ? n : a.N - 1) + s * a.N;
    wp[s] = static_cast<const uint8_t*>(a.weight) + n * a.ldw * EB;
  }
  const uint8_t* xp[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    int64_t m = mbase + R * j + ri;
    m = m < a.M ? m : a.M - 1;
    xp[j] = static_cast<const uint8_t*>(a.x) + m * a.ldx * EB;
  }
  const int steps = (kfull + STEP - 1) / STEP;
  const int per = (steps + waves - 1) / waves;
  const int s0 = wave * per;
  const int s1 = s0 + per < steps ? s0 + per : steps;
  const int off = (ci * 4 + q) * 16;  // this lane's 16 bytes of a step

  // U steps in flight while the U before them are multiplied.  Every load is
  // unconditional: past the wave's range or the row's last whole 16 bytes it
  // reads the row's first and is cleared.  (kfull 0: no row has 16 bytes.)
  u32x4 w0[U][NS], x0[U][MT], w1[U][NS], x1[U][MT];
  auto load = [&](u32x4 (&w)[U][NS], u32x4 (&x)[U][MT], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int o = (s + u) * STEP + off;
      const int oc = s + u < s1 && o < kfull ? o : 0;
#pragma unroll
      for (int i = 0; i < NS; ++i) w[u][i] = ld16_any(wp[i] + oc);
#pragma unroll
      for (int j = 0; j < MT; ++j) x[u][j] = ld16_any(xp[j] + oc);
    }
  };

  // e4m3: scales of the strips' rows and of the group's rows of x, all K blocks:
  // s_ws[kb][strip][row], s_xs[kb][group row]; block `kblocks` of zeros is for chunks
  // that were cleared (0 times an infinite scale would be NaN)
  const int kblocks = FP8 ? static_cast<int>(a.K / 128) : 0;
  float* s_ws = lds;
  float* s_xs = s_ws + (FP8 ? (kblocks + 1) * NS * R : 0);
  float* red = s_xs + (FP8 ? (kblocks + 1) * MT * R : 0);

  const bool any = s0 < s1;  // uniform per wave
  if (any) load(w0, x0, s0);
  if constexpr (FP8) {
    for (int i = tid; i < (kblocks + 1) * NS * R; i += blockDim.x) {
      const int kb = i / (NS * R), s = (i / R) % NS, r = i % R;
      int64_t n = n0 + r;
      n = (n < a.N ? n : a.N - 1) + s * a.N;
      s_ws[i] = kb < kblocks ? a.weight_scale[(n / 128) * a.weight_scale_row + kb * a.weight_scale_blk]
                             : 0.f;
    }
    for (int i = tid; i < (kblocks + 1) * MT * R; i += blockDim.x) {
      const int kb = i / (MT * R);
      int64_t m = mbase + i % (MT * R);
      m = m < a.M ? m : a.M - 1;
      s_xs[i] = kb < kblocks ? a.x_scale[m * a.x_scale_row + kb * a.x_scale_blk] : 0.f;
    }
    __syncthreads();
  }

  f32x4 acc[NS][MT];
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the lane's results: rows 4 q .. 4 q + 3 of the 16 (chunk co, strip rows
  // ro .. ro + 3), column l16 (chunk ci, row of x ri)
  const int co = (4 * q) / R, ro = (4 * q) % R;

  auto product = [&](const u32x4 (&w)[NS], const u32x4 (&x)[MT], int s) __attribute__((always_inline)) {
    if constexpr (FP8) {
      uint4 xb[MT][2];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        xb[j][0] = fp8x8_to16<false, false>(make_uint2(x[j].x, x[j].y));
        xb[j][1] = fp8x8_to16<false, false>(make_uint2(x[j].z, x[j].w));
      }
      const int kr = (s * STEP + co * 64) / 128;  // K block of the lane's results
      const int kb = s < s1 && kr < kblocks ? kr : kblocks;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const uint4 wa = fp8x8_to16<false, false>(make_uint2(w[i].x, w[i].y));
        const uint4 wb = fp8x8_to16<false, false>(make_uint2(w[i].z, w[i].w));
        const f32x4 ws = *reinterpret_cast<const f32x4*>(s_ws + (kb * NS + i) * R + ro);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          f32x4 d = {0.f, 0.f, 0.f, 0.f};
          d = mfma16_16x16x32<false>(wa, xb[j][0], d);
          d = mfma16_16x16x32<false>(wb, xb[j][1], d);
          const float xs = s_xs[kb * MT * R + j * R + ri];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] += d[r] * (xs * ws[r]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j)
          acc[i][j] = mfma16_16x16x32<F16>(as4(w[i]), as4(x[j]), acc[i][j]);
    }
  };
  auto compute = [&](u32x4 (&w)[U][NS], u32x4 (&x)[U][MT], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t keep = s + u < s1 && (s + u) * STEP + off < kfull ? ~0u : 0u;
#pragma unroll
      for (int i = 0; i < NS; ++i) w[u][i] &= keep;
#pragma unroll
      for (int j = 0; j < MT; ++j) x[u][j] &= keep;
      product(w[u], x[u], s + u);
    }
  };
  // GUARD: no loads behind the range.  Narrow gated e4m3 strips gain (us, kernels
  // alone, without / with: 3 x 7168 x 4096 15.0 / 11.1, 4 x 4096 x 4096 13.7 / 8.2, 4 x
  // 2048 x 4096 7.4 / 6.2, 1 x 2048 x 1536 5.5 / 4.7, 4 x 7168 x 2048 8.5 / 8.5; 2 x 2816 x
  // 2560 loses, 6.8 / 7.4); the branches cost the others more than the loads, which
  // hit the caches (bf16 1 x 7168 x 256 5.3 -> 5.7, 8 x 7168 x 4096 gated 16.1 -> 18.1).
  constexpr bool GUARD = FP8 && GATED && R * MT == 4;
  if (any) {
    for (int s = s0; s < s1; s += 2 * U) {
      if (!GUARD || s + U < s1) load(w1, x1, s + U);
      compute(w0, x0, s);
      if (GUARD && s + U >= s1) break;
      if (!GUARD || s + 2 * U < s1) load(w0, x0, s + 2 * U);
      compute(w1, x1, s + U);
    }
  }
  // the last K % 8 values of 16-bit rows: wave 0, element by element
  if constexpr (!FP8) {
    if (kfull < kbytes && wave == 0) {
      auto tail = [&](const uint8_t* row) __attribute__((always_inline)) {
        uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 7; ++k)
          if (ci == 0 && q == 0 && kfull + 2 * k < kbytes)
            v[k >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + kfull + 2 * k))
                         << (16 * (k & 1));
        return u32x4{v[0], v[1], v[2], v[3]};
      };
      u32x4 w[NS], x[MT];
#pragma unroll
      for (int i = 0; i < NS; ++i) w[i] = tail(wp[i]);
#pragma unroll
      for (int j = 0; j < MT; ++j) x[j] = tail(xp[j]);
      product(w, x, 0);
    }
  }

  // red[wave][strip][group][chunk][row of x][strip row]
  constexpr int TILE = C * R * R;
  if (co == ci) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j)
        *reinterpret_cast<f32x4*>(red + ((wave * NS + i) * MT + j) * TILE + (ci * R + ri) * R + ro) =
            acc[i][j];
  }
  __syncthreads();
  for (int o = tid; o < MT * R * R; o += blockDim.x) {
    const int r = o % R, mr = (o / R) % R, j = o / (R * R);
    const int64_t n = n0 + r, m = mbase + R * j + mr;
    if (n >= a.N || m >= a.M) continue;
    float z = 0.f, u = 0.f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float* p = red + (w * NS * MT + j) * TILE + (c * R + mr) * R + r;
        z += p[0];
        if constexpr (GATED) u += p[MT * TILE];
      }
    st_any(a.out, a.out_dtype, m * a.ldo + n, lin_value(a, m, n, z, u));
  }
}

template <bool FP8, bool F16, bool GATED, int R, int MT, int U>
int launch(const LinArgs& a, int waves, hipStream_t st) {
  constexpr int NS = GATED ? 2 : 1;
  const int64_t blocks = FP8 ? a.K / 128 + 1 : 0;
  // at most 48 KiB of scales (linear_skinny_takes), a block of zeros and 8 KiB of sums
  const size_t lds = 4 * (blocks * (NS + MT) * R + static_cast<size_t>(waves) * NS * MT * 16 * R);
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, R)), static_cast<unsigned>(cdiv(a.M, R * MT)));
  linear_skinny_kernel<FP8, F16, GATED, R, MT, U><<<grid, dim3(64 * waves), lds, st>>>(a);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

// Strip height and waves, from sweeps over all of them at 1 to 48 rows of the
// products below (here and above: rows x K x weight rows, both halves of a gated
// weight counted).  Strips of 4 or 8 rows win while strips of 16 leave CUs
// without work (16-bit, 8 rows, 7168 x 4096 gated: 4-row strips 16.0 us, 16-row
// 24.0); strips of 16 read x a quarter as often (4 x 7168 x 7168 23.8 against
// 26.0, 16 x 4096 x 4096 12.2 against 15.1) and stage e4m3 scales once per 16 rows
// (4 x 2048 x 7168 7.6 against 8.5).  More waves per strip shorten the walk over a
// long K and lengthen the sum at its end (1 x 7168 x 7168 with 1 / 2 / 4 waves 21.0 /
// 21.9 / 23.4, e4m3 1 x 7168 x 4096 gated 19.1 / 13.9 / 11.7, before GUARD).
template <bool FP8, bool F16, bool GATED>
int launch_rows(const LinArgs& a, hipStream_t st) {
  const bool few = a.N <= 2048;  // at most 128 strips of 16
  if constexpr (FP8) {
    const bool lng = a.K >= 4096;
    if (a.M <= 4 && few) return launch<FP8, F16, GATED, 4, 1, 4>(a, lng ? 4 : 2, st);
    if (a.M <= 8 && few && lng) return launch<FP8, F16, GATED, 4, 2, 4>(a, 4, st);
    if (few && lng) return launch<FP8, F16, GATED, 8, 2, 4>(a, 4, st);
    return launch<FP8, F16, GATED, 16, 1, 4>(a, 4, st);
  } else {
    if (a.M == 1 || (a.M <= 4 && a.N < 4096))
      return launch<FP8, F16, GATED, 4, 1, 4>(a, few ? 2 : 1, st);
    if (a.M <= 8 && few) return launch<FP8, F16, GATED, 4, 2, 4>(a, a.N <= 1024 ? 2 : 1, st);
    if (few && (a.M <= 16 || a.N <= 512)) return launch<FP8, F16, GATED, 8, 2, 4>(a, 2, st);
    return launch<FP8, F16, GATED, 16, 1, 4>(a, a.N <= 5120 && a.M <= 16 ? 4 : 2, st);
  }
}

}  // namespace

// Rows of x that the stream takes.  Its waves walk K, so a long K and many rows
// go to the tiles, which split it (skinny / tile us: 8 x 7168 x 2048 11.9 / 12.1 e4m3,
// 13.6 / 13.4 bf16; 16 x 7168 x 256 11.9 / 9.5, 12.1 / 10.3; 16 x 7168 x 7168 22.9 / 18.0,
// 33.4 / 24.4; 16 x 4096 x 4096 9.2 / 12.1, 12.2 / 13.5); e4m3 products of large
// weights from 5 rows on (8 x 7168 x 4096 gated 16.5 / 13.7, 4 rows 10.9 / 13.6).  Past 16
// rows it streams the weight once per 16: for weights that leave the tiles
// short of work (32 x 2048 x 1536 gated 7.0 / 9.6 and 9.7 / 12.0, 61 x 2048 x
// 1536 8.1 / 9.8 and 10.8 / 10.4; 32 x 2816 x 2816 11.9 / 9.9 and 15.2 / 12.4).
// Rows that the tiles cannot fetch (`tile` false): any K, and small weights.
bool linear_skinny_takes(const LinArgs& a, bool tile) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  if (fp8 && (a.K / 128) * 48 * 4 > kScaleBytes) return false;  // scales beyond their LDS
  const int64_t weight = lin_rows(a) * a.K;
  if (!tile) return a.M <= 16 || (a.M <= 64 && weight <= (int64_t(4) << 20));
  if (a.K > 4096) return a.M <= (fp8 && weight > (int64_t(16) << 20) ? 4 : 8);
  return a.M <= 16 || (a.M <= 64 && cdiv(a.M, 16) * weight <= (int64_t(12) << 20));
}

int launch_linear_skinny(const LinArgs& a, hipStream_t st) {
  const bool g = lin_gated(a.activation);
  if (a.x_dtype == MI355MOE_FP8E4M3)
    return g ? launch_rows<true, false, true>(a, st) : launch_rows<true, false, false>(a, st);
  if (a.x_dtype == MI355MOE_F16)
    return g ? launch_rows<false, true, true>(a, st) : launch_rows<false, true, false>(a, st);
  return g ? launch_rows<false, false, true>(a, st) : launch_rows<false, false, false>(a, st);
}

}  // namespace mi355
