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
// QUANT: x is one 16-bit row; every workgroup makes its int8 codes itself, into LDS, while
// its first weights are on their way.
//
// e4m3 operands are converted to bf16 (exact) as they arrive; each K step's
// product is multiplied by its blocks' scales, held in LDS.
#include "int8_quant.h"

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

// The row's scale and codes (K % 16 == 0): each of 256 threads holds 4 chunks of 8 columns
// at most.
constexpr int kQuantChunks = 4;
__device__ __forceinline__ void load_row(const LinArgs& a, int waves, uint4 (&row)[kQuantChunks]) {
#pragma unroll
  for (int c = 0; c < kQuantChunks; ++c) {
    const int64_t i = static_cast<int64_t>(c * 64 * waves + threadIdx.x) * 8;
    row[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + (i < a.K ? i : 0));
  }
}
template <typename E>
__device__ __forceinline__ void quantise_row(const LinArgs& a, int waves, const uint4 (&row)[kQuantChunks],
                                             float* s_scale, uint8_t* s_code) {
  __shared__ uint32_t s_top[4];
  const int tid = threadIdx.x, threads = 64 * waves;
  float f[kQuantChunks][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < kQuantChunks; ++c) {
    unpack_row8<E>(row[c], f[c]);  // (chunks past the row repeat its first)
    const uint32_t u = top8(f[c]);
    top = u > top ? u : top;
  }
  top = wave_top(top);
  if ((tid & 63) == 0) s_top[tid >> 6] = top;
  __syncthreads();
  for (int w = 0; w < waves; ++w) top = s_top[w] > top ? s_top[w] : top;
  const float s = scale_of(top);
  if (tid == 0) *s_scale = s;
#pragma unroll
  for (int c = 0; c < kQuantChunks; ++c) {
    const int64_t i = static_cast<int64_t>(c * threads + tid) * 8;
    if (i < a.K) *reinterpret_cast<uint2*>(s_code + i) = codes8(f[c], s);
  }
  __syncthreads();
}

template <int KIND, bool GATED, int R, int MT, int U, bool QUANT>
__global__ __launch_bounds__(256) void linear_skinny_kernel(const LinArgs a) {
  constexpr int C = 16 / R;
  constexpr int STEP = C * 64;                // bytes of a row per K step
  constexpr int NS = GATED ? 2 : 1;           // strips: the gate's, the factor's
  constexpr bool FP8 = KIND == K_FP8, I8 = KIND == K_I8;
  using Sum = typename SumVec<KIND, 4>::T;
  using S = std::conditional_t<I8, int, float>;
  constexpr int EB = kind_bytes(KIND);
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = static_cast<int>(blockDim.x) >> 6;
  const int l16 = lane & 15, q = lane >> 4;
  const int ri = l16 % R, ci = l16 / R;
  static_assert(!QUANT || (I8 && MT == 1), "operands");
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
    xp[j] = static_cast<const uint8_t*>(a.x) + m * a.ldx * EB;  // (QUANT: not read)
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
      if constexpr (!QUANT) {
#pragma unroll
        for (int j = 0; j < MT; ++j) x[u][j] = ld16_any(xp[j] + oc);
      }
    }
  };

  // e4m3: scales of the strips' rows and of the group's rows of x, all K blocks:
  // s_ws[kb][strip][row], s_xs[kb][group row]; block `kblocks` of zeros is for chunks
  // that were cleared (0 times an infinite scale would be NaN)
  const int kblocks = FP8 ? static_cast<int>(a.K / 128) : 0;
  float* s_ws = lds;
  float* s_xs = s_ws + (FP8 ? (kblocks + 1) * NS * R : 0);
  S* red = reinterpret_cast<S*>(s_xs + (FP8 ? (kblocks + 1) * MT * R : 0));

  const bool any = s0 < s1;  // uniform per wave
  // QUANT: the row's loads before the weights' (loads end in order), which are on their way
  // while the row's scale and then its codes are made
  [[maybe_unused]] uint4 row[kQuantChunks];
  if constexpr (QUANT) {
    load_row(a, waves, row);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (any) {
    load(w0, x0, s0);
    if constexpr (QUANT) {
      load(w1, x1, s0 + U);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  float* s_row = lds;
  uint8_t* s_code = reinterpret_cast<uint8_t*>(lds + 4);
  if constexpr (QUANT) {
    red = reinterpret_cast<S*>(s_code + a.K);
    if (a.x_dtype == MI355MOE_F16) quantise_row<F16>(a, waves, row, s_row, s_code);
    else quantise_row<BF16>(a, waves, row, s_row, s_code);
  }
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

  Sum acc[NS][MT];
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = Sum{0, 0, 0, 0};
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
          acc[i][j] = mfma_16x16<KIND>(as4(w[i]), as4(x[j]), acc[i][j]);
    }
  };
  auto compute = [&](u32x4 (&w)[U][NS], u32x4 (&x)[U][MT], int s) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t keep = s + u < s1 && (s + u) * STEP + off < kfull ? ~0u : 0u;
#pragma unroll
      for (int i = 0; i < NS; ++i) w[u][i] &= keep;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if constexpr (QUANT) {  // (every row of the group is the one; cleared weights need no codes)
          x[u][j] = *reinterpret_cast<const u32x4*>(s_code + (keep ? (s + u) * STEP + off : 0));
        } else {
          x[u][j] &= keep;
        }
      }
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
      if (QUANT ? s != s0 : !GUARD || s + U < s1) load(w1, x1, s + U);
      compute(w0, x0, s);
      if (GUARD && s + U >= s1) break;
      if (!GUARD || s + 2 * U < s1) load(w0, x0, s + 2 * U);
      compute(w1, x1, s + U);
    }
  }
  // the last K % 8 values of 16-bit rows, K % 16 of int8 ones: wave 0, element by element
  if constexpr (!FP8) {
    if (kfull < kbytes && wave == 0) {
      auto tail = [&](const uint8_t* row) __attribute__((always_inline)) {
        uint32_t v[4] = {0, 0, 0, 0};
        if constexpr (I8) {
#pragma unroll
          for (int k = 0; k < 15; ++k)
            if (ci == 0 && q == 0 && kfull + k < kbytes)
              v[k >> 2] |= static_cast<uint32_t>(row[kfull + k]) << (8 * (k & 3));
        } else {
#pragma unroll
          for (int k = 0; k < 7; ++k)
            if (ci == 0 && q == 0 && kfull + 2 * k < kbytes)
              v[k >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + kfull + 2 * k))
                           << (16 * (k & 1));
        }
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
        *reinterpret_cast<Sum*>(red + ((wave * NS + i) * MT + j) * TILE + (ci * R + ri) * R + ro) =
            acc[i][j];
  }
  __syncthreads();
  for (int o = tid; o < MT * R * R; o += blockDim.x) {
    const int r = o % R, mr = (o / R) % R, j = o / (R * R);
    const int64_t n = n0 + r, m = mbase + R * j + mr;
    if (n >= a.N || m >= a.M) continue;
    S z = 0, u = 0;
    for (int w = 0; w < waves; ++w)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const S* p = red + (w * NS * MT + j) * TILE + (c * R + mr) * R + r;
        z += p[0];
        if constexpr (GATED) u += p[MT * TILE];
      }
    float y;
    if constexpr (I8) y = lin_value_i32(a, m, n, QUANT ? *s_row : x_scale_of(a, m), z, u);
    else y = lin_value(a, m, n, z, u);
    st_any(a.out, a.out_dtype, m * a.ldo + n, y);
  }
}

template <int KIND, bool GATED, int R, int MT, int U, bool QUANT = false>
int launch(const LinArgs& a, int waves, hipStream_t st) {
  constexpr int NS = GATED ? 2 : 1;
  const int64_t blocks = KIND == K_FP8 ? a.K / 128 + 1 : 0;
  // QUANT: the row's scale and codes (K up to 8192: 8 KiB);
  // at most 48 KiB of scales (linear_skinny_takes), a block of zeros and 8 KiB of sums
  const size_t lds = (QUANT ? 16 + a.K : 0) + 4 * (blocks * (NS + MT) * R + static_cast<size_t>(waves) * NS * MT * 16 * R);
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, R)), static_cast<unsigned>(cdiv(a.M, R * MT)));
  linear_skinny_kernel<KIND, GATED, R, MT, U, QUANT><<<grid, dim3(64 * waves), lds, st>>>(a);
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
template <int KIND, bool GATED>
int launch_rows(const LinArgs& a, hipStream_t st) {
  const bool few = a.N <= 2048;  // at most 128 strips of 16
  if constexpr (KIND == K_I8) {
    // Two steps ahead (U = 2) are enough for bytes, and shorter to fill (1 x 4096 x 4096 6.4
    // us against 7.0 with four, 4 x 7168 x 4096 gated 10.0 / 10.6, 8 x 4096 x 4096 7.7 / 8.0,
    // 16 x 4096 x 4096 8.3 / 8.9, 16 x 2048 x 1536 gated 5.3 / 5.7).
    if (a.x_dtype != MI355MOE_I8) return launch<KIND, GATED, 4, 1, 2, true>(a, 4, st);
    // One row over a long K: four waves to a strip where there are not many of them (us, two /
    // four: 1 x 7168 x 7168 14.1 / 13.1, 1 x 8192 x 8192 gated 17.0 / 15.7, 1 x 2880 x 5760 7.2 / 6.5,
    // 1 x 4096 x 4096 6.2 / 6.2, but 1 x 2048 x 7168 5.9 / 7.6, 1 x 4096 x 22016 gated 21.0 / 22.6,
    // 4 x 7168 x 4096 gated 10.2 / 10.4).
    const bool four = a.M == 1 && a.K >= 2880 && lin_rows(a) <= 8192;
    if (a.M <= 4) return launch<KIND, GATED, 4, 1, 2>(a, four ? 4 : 2, st);
    if (a.M <= 16 && few) return launch<KIND, GATED, 8, 2, 2>(a, 2, st);
    return launch<KIND, GATED, 16, 1, 2>(a, 4, st);
  } else if constexpr (KIND == K_FP8) {
    const bool lng = a.K >= 4096;
    if (a.M <= 4 && few) return launch<KIND, GATED, 4, 1, 4>(a, lng ? 4 : 2, st);
    if (a.M <= 8 && few && lng) return launch<KIND, GATED, 4, 2, 4>(a, 4, st);
    if (few && lng) return launch<KIND, GATED, 8, 2, 4>(a, 4, st);
    return launch<KIND, GATED, 16, 1, 4>(a, 4, st);
  } else {
    if (a.M == 1 || (a.M <= 4 && a.N < 4096))
      return launch<KIND, GATED, 4, 1, 4>(a, few ? 2 : 1, st);
    if (a.M <= 8 && few) return launch<KIND, GATED, 4, 2, 4>(a, a.N <= 1024 ? 2 : 1, st);
    if (few && (a.M <= 16 || a.N <= 512)) return launch<KIND, GATED, 8, 2, 4>(a, 2, st);
    return launch<KIND, GATED, 16, 1, 4>(a, a.N <= 5120 && a.M <= 16 ? 4 : 2, st);
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
// int8, whose tiles' sums of a split cost as much and whose stream is half as long, streams more
// (16 x 7168 x 4096 gated 12.2 / 14.2, 16 x 7168 x 7168 20.2 / 17.3, 32 x 7168 x 4096 gated 14.7 /
// 15.4, 61 x 2880 x 2880 10.7 / 14.4, 61 x 2048 x 1536 gated 6.5 / 9.9, 61 x 4096 x 4096 20.2 / 13.0;
// a short K leaves it little to hide its start behind: 32 x 512 x 4096 5.8 / 5.3).
// Rows that the tiles cannot fetch (`tile` false): any K, and small weights.
bool linear_skinny_takes(const LinArgs& a, bool tile) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  if (fp8 && (a.K / 128) * 48 * 4 > kScaleBytes) return false;  // scales beyond their LDS
  const int64_t weight = lin_rows(a) * a.K;
  if (!tile) return a.M <= 16 || (a.M <= 64 && weight <= (int64_t(4) << 20));
  if (a.x_dtype == MI355MOE_I8)
    return a.M <= 8 || (a.M <= 16 && weight <= (int64_t(32) << 20)) ||
           (a.M <= 64 && a.K >= 1024 && cdiv(a.M, 16) * weight <= (int64_t(32) << 20));
  if (a.K > 4096) return a.M <= (fp8 && weight > (int64_t(16) << 20) ? 4 : 8);
  return a.M <= 16 || (a.M <= 64 && cdiv(a.M, 16) * weight <= (int64_t(12) << 20));
}

// x that the stream quantises itself: one row at a multiple of 16 bytes.  A launch less, but
// each workgroup of 4 weight rows quantises it again, so up to 4 of them per CU (both ways in a
// graph, us: 1 x 7168 x 4096 gated 11.7 / 12.7, 1 x 8192 x 8192 gated 16.0 / 18.9, 1 x 2048 x 1536
// gated 5.6 / 7.1, 1 x 7168 x 256 6.3 / 7.8, 1 x 4096 x 4096 8.2 / 8.9, but 1 x 4096 x 6144 10.8 /
// 10.1, 1 x 4096 x 14336 17.7 / 15.8).  The row's loads go first: behind the weights' its codes
// would wait for them (1 x 8192 x 8192 gated 18.7, with fewer weights ahead 19.3).
bool linear_skinny_quantises(const LinArgs& a) {
  return a.M == 1 && a.N <= 4096 && a.K % 16 == 0 && a.K <= 8 * 256 * kQuantChunks &&
         (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
}

int launch_linear_skinny(const LinArgs& a, hipStream_t st) {
  const bool g = lin_gated(a.activation);
  if (a.x_dtype == MI355MOE_FP8E4M3)
    return g ? launch_rows<K_FP8, true>(a, st) : launch_rows<K_FP8, false>(a, st);
  if (a.x_dtype == MI355MOE_I8 || a.weight_dtype == MI355MOE_I8)
    return g ? launch_rows<K_I8, true>(a, st) : launch_rows<K_I8, false>(a, st);
  if (a.x_dtype == MI355MOE_F16)
    return g ? launch_rows<K_F16, true>(a, st) : launch_rows<K_F16, false>(a, st);
  return g ? launch_rows<K_BF16, true>(a, st) : launch_rows<K_BF16, false>(a, st);
}

}  // namespace mi355
