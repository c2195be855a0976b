// Tiles of a matrix product on operands that direct copies to LDS can fetch: BI x BJ
// outputs, stages of 128 bytes of each operand's row.  out[i, j] = sum_r q(i, r) p(j, r):
// a linear's x and weight lie along r (int8 and 16-bit operands); the products of a
// backward pass have p, and maybe q, across it (16-bit operands).
//
// LDS.  A ring of NSTAGE stages.  An operand along r: the rows' 128 bytes one after the
// other, 16-byte chunk c of row i at slot c ^ swz(i), so that the 16 rows of a quarter
// of a fragment read cover all 64 banks once.  An operand across r: 64 rows of the
// tile's columns as they are; the transposing LDS read gives each lane 4 r of its
// column, two reads a fragment.  A group of 16 lanes reads 32 bytes of 4 rows, 32 lanes
// 64 bytes of them, so chunks of consecutive rows are moved by 64 bytes (cross_swz): the
// 4 rows then cover all 64 banks once.
//
// 32x32x16 (int8: 32x32x32) MFMAs, p as the A operand, so that a lane's sums are
// consecutive columns of one row of out; four steps per stage, the next step's fragments
// read while this one's MFMAs run; the barrier that publishes the next stage sits before
// the last step.  Rows and columns past the edges repeat the last ones and are not
// stored; the last stage's r past R are cleared in LDS.
//
// The epilogue takes the sums from the registers: a swap of half waves gives each lane 8
// consecutive columns, one of 16-lane groups makes a wave's 16-byte stores 16 rows x 64 bytes
// (of 16-bit outputs); the scales of int8 and the biases wait in LDS, residuals are loaded one row of tiles ahead.  No LDS
// of the ring is needed for that, so a workgroup takes tile after tile, and the next one's
// first stages are on their way meanwhile.
#pragma once

#include "linear.h"
#include "product.h"
#include "tile.h"
#include "tile_walk.h"

namespace mi355 {

constexpr int GSB = 128;         // bytes of a stage along r
__device__ __forceinline__ int gswz(int r) { return (r >> 1) & 7; }
// across r: chunk c of row r is at slot c ^ cross_swz<chunks of a row>(r): 64 bytes times r & 3
// where rows start at the same banks (multiples of 256 bytes), 64 times r / 2 where every
// other one does; rows of 192 bytes are 64 apart as they are
template <int CH>
__device__ __forceinline__ int cross_swz(int r) {
  static_assert(CH % 8 == 0 || CH == 12, "rows");
  return CH % 16 == 0 ? (r & 3) << 2 : CH % 8 == 0 ? ((r >> 1) & 1) << 2 : 0;
}

// What a tile does with its sums: E_RAW, as they are to a.out + split M N (float, int8:
// int32); E_PLAIN, rounded to the operands' type; E_LINEAR, a linear's epilogue; E_KEEP, the
// same of a gated one, and the sums with their biases to a.z.
enum { E_RAW = 0, E_PLAIN = 1, E_LINEAR = 2, E_KEEP = 3 };

// 8 sums of consecutive columns in each lane: lo holds columns 4 h .. 4 h + 3, hi 8 + 4 h ..;
// lane half h gets columns 8 h .. 8 h + 7.
template <typename V>
__device__ __forceinline__ void gather8(const V& acc, int g, uint32_t (&o)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const auto lo = acc[8 * g + k], hi = acc[8 * g + 4 + k];
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, lo),
                                                    __builtin_bit_cast(uint32_t, hi), false, false);
    o[k] = r[0];
    o[4 + k] = r[1];
  }
}

// 16 bytes to or from an address of any alignment (gfx950's global accesses need none)
typedef uint32_t any16_t __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void put16(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *static_cast<any16_t*>(p) = any16_t{a, b, c, d};
}

// Two runs of 8 columns, a of columns 8 h .. and b of 16 + 8 h .. of row l32: a swap of
// 16-lane groups gives runs whose lanes cover 32 columns of 16 rows (64 bytes of 16-bit
// outputs instead of 32): columns 16 (g & 1) + 8 (g / 2) .. of row t16 in a, of row
// 16 + t16 in b (g, t16: the lane's group of 16 and its place there).  Its own inverse.
template <int N>
__device__ __forceinline__ void pair16(uint32_t (&a)[N], uint32_t (&b)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const auto r = __builtin_amdgcn_permlane16_swap(a[k], b[k], false, false);
    a[k] = r[0];
    b[k] = r[1];
  }
}

// (two workgroups to a CU where their LDS fits: at most 256 registers then)
constexpr int gemm_waves_per_simd(int waves, int bi, int bj, int stages) {
  return (waves / 4) * (2 * (stages * (bi + bj) * GSB + 4 * (2 * bj + bi)) <= 160 * 1024 ? 2 : 1);
}
// floats of biases and scales behind the ring
constexpr int gemm_side(int kind, int epi, int bi, int bj) {
  return epi == E_LINEAR || epi == E_KEEP ? bj + (kind == K_I8 ? bi + bj : 0) : 0;
}
template <int KIND, bool TQ, bool TP, bool GATED, int EPI, int BI, int BJ, int WI, int WJ, int NSTAGE>
__global__ __launch_bounds__(64 * WI * WJ, gemm_waves_per_simd(WI * WJ, BI, BJ, NSTAGE)) void gemm_tile_kernel(
    const LinArgs a, int tiles_i, int tiles_j, int splits, int stages_per_split) {
  constexpr int BYTES = NSTAGE * (BI + BJ) * GSB + 4 * gemm_side(KIND, EPI, BI, BJ);
  static_assert(BYTES <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[BYTES];
  XcdWalk walk(tiles_i * tiles_j * splits, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
#include "gemm_tile_body.h"
}

// A choice of tiles.  us: time of one stage on every CU at once, round: of the rest of a
// round of tiles (first copies, epilogue); per_cu: workgroups of the tile that a CU holds.
enum TileShape {
  G256X256, G256X128, G128X256, G192X192, G192X128, G128X192, G128X128X2, G128X128, G96X128, G64X128X2, G64X64X3
};
struct TileSpec {
  TileShape shape;
  int bi, bj, per_cu;
  float us, round;
};
// a shape's waves take the same columns of both halves of a gated weight, in 32s; G128X192 is
// for these alone
constexpr bool gates_of(TileShape s) {
  return s != G192X192 && s != G192X128 && s != G96X128 && s != G64X64X3;
}
struct TilePlan {
  TileShape shape;
  int splits, per;  // stages per split
};
// The tile and the split of r with the least estimated time for I x `rows` (of p) outputs (J
// columns where gates halve them) of `nk` stages: rounds of the grid over the CUs, and for a
// split the partial sums written and read at 3.5 TB/s and a second launch.
// (A call prices its tiles more than once, and small steps wait for the host: about 0.5 us here.)
template <int N>
TilePlan gemm_plan(const TileSpec (&tiles)[N], int64_t I, int64_t J, int64_t rows, int nk) {
  constexpr int kMaxSplits = 16, kMaxSplitTiles = 1 << 16;
  int splits[kMaxSplits], pers[kMaxSplits], count = 0;
  for (int s = 1; s <= kMaxSplits; ++s) {
    const int per = (nk + s - 1) / s;
    if (s > 1 && per < 4) break;
    if (s > 1 && (nk + per - 1) / per != s) continue;
    splits[count] = s;
    pers[count++] = per;
  }
  TilePlan best{};
  double best_us = -1;
  for (const TileSpec& c : tiles) {
    const bool halves = rows != J;  // gates; a split product has none: all rows of p
    const int64_t ti = cdiv(I, c.bi), whole = ti * cdiv(rows, c.bj);
    const int64_t gated = halves ? ti * cdiv(J, c.bj / 2) : whole;
    const int64_t most = 256 * c.per_cu;
    // (workgroups that share a CU share its LDS copies: alone, 128 x 128 takes 0.62 us a stage
    // against 0.97 two together, 64 x 64 0.33 against 0.50 and 0.70)
    const double alone = c.us / (1 + 0.6 * (c.per_cu - 1));
    for (int k = 0; k < count; ++k) {
      const int s = splits[k];
      const bool gates = halves && s == 1;
      if (gates ? !gates_of(c.shape) : c.shape == G128X192) continue;
      const int64_t n = gates ? gated : whole * s;
      if (s > 1 && n > kMaxSplitTiles) break;
      double us;
      if (n < most) us = alone * (1 + 0.6 * static_cast<double>((n + 255) / 256 - 1)) * pers[k] + c.round;
      else us = static_cast<double>((n + most - 1) / most) * (c.us * pers[k] + c.round);
      // (3.1 rather than 4: 61 x 4096 x 6144 in int8 from HBM 17.7 -> 15.8 us, from a cache 13.7 -> 13.9;
      // dx 128 x 4096 x 7168 27.6 -> 26.0; at 3 200 x 2048 x 1536 gated would lose, 10.6 / 11.4)
      if (s > 1) us += 3.1 + 2.0 * s * I * rows * 4 / 3.5e6;
      if (best_us < 0 || us < best_us) {
        best = {c.shape, s, pers[k]};
        best_us = us;
      }
    }
  }
  return best;
}

template <int KIND, bool TQ, bool TP, bool GATED, int EPI, int BI, int BJ, int WI, int WJ, int NSTAGE>
int launch_gemm(const LinArgs& a, const TilePlan& p, int per_cu, hipStream_t st) {
  const int64_t ti = cdiv(a.M, BI), tj = cdiv(a.N, GATED ? BJ / 2 : BJ), total = ti * tj * p.splits;
  const int64_t most = 256 * per_cu;  // a workgroup takes the tiles this far apart in its XCD's range
  const dim3 grid(static_cast<unsigned>(total < most ? cdiv(total, 8) * 8 : most));
  gemm_tile_kernel<KIND, TQ, TP, GATED, EPI, BI, BJ, WI, WJ, NSTAGE>
      <<<grid, dim3(64 * WI * WJ), 0, st>>>(a, static_cast<int>(ti), static_cast<int>(tj), p.splits, p.per);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}
// Waves and stages.  Where a CU holds one workgroup, tiles with sides of 128 and 256 have 8 waves,
// which hide each other's latency; those with a side of 96 or 192, for the fill of the CUs, have 4
// (more were not measured).  256 x 256 in 8 waves of 128 x 64 against 4 of 128 x 128, which read a
// third less from LDS (in turn, us: int8 8192 x 7168 x 4096 gated 214 / 232, kept 421 / 447, dx 8192
// x 4096 x 7168 412 / 433, dW 4096 x 8192 x 7168 405 / 413); 128 x 128 in 8 and 4 (int8 1003 x 2880
// x 2880 21.0 / 23.9).  Small tiles share a CU: 64 x 128 with two workgroups of three stages against
// one of four (dW 2048 x 512 x 4096 16.6 / 21.9, int8 1003 x 2880 x 2880 22.9 / 28.9), 64 x 64 three
// of three, two of four and one of eight (dx 512 x 2048 x 4096 16.5 / 17.0 / 25.7).  The gated 256 x
// 256 epilogues, int8 and kept, hold more than the 256 registers and spill 78 and 43 of them around
// a tile (220 and 176 bytes of scratch a lane, none on the way through full stages); a stage still
// takes 1.78 us where two of 128 x 256, which do not spill, take 1.96.  No other tile spills.
template <int KIND, bool TQ, bool TP, bool GATED, int EPI>
int launch_gemm_shape(const LinArgs& a, const TilePlan& p, hipStream_t st) {
  switch (p.shape) {
    case G256X256:
      // (the sums and an ungated linear's epilogue leave too few registers)
      if constexpr (EPI != E_LINEAR || GATED)
        return launch_gemm<KIND, TQ, TP, GATED, EPI, 256, 256, 2, 4, 2>(a, p, 1, st);
      break;
    case G256X128: return launch_gemm<KIND, TQ, TP, GATED, EPI, 256, 128, 4, 2, 3>(a, p, 1, st);
    case G128X256: return launch_gemm<KIND, TQ, TP, GATED, EPI, 128, 256, 2, 4, 3>(a, p, 1, st);
    case G192X192:
      if constexpr (!GATED && KIND != K_I8)  // (int8: no table has it, its epilogue spills)
        return launch_gemm<KIND, TQ, TP, GATED, EPI, 192, 192, 2, 2, 3>(a, p, 1, st);
      break;
    case G192X128:
      if constexpr (!GATED) return launch_gemm<KIND, TQ, TP, GATED, EPI, 192, 128, 2, 2, 3>(a, p, 1, st);
      break;
    case G96X128:
      if constexpr (!GATED) return launch_gemm<KIND, TQ, TP, GATED, EPI, 96, 128, 1, 4, 4>(a, p, 1, st);
      break;
    case G128X192:
      if constexpr (GATED) return launch_gemm<KIND, TQ, TP, GATED, EPI, 128, 192, 4, 1, 3>(a, p, 1, st);
      break;
    case G128X128X2: return launch_gemm<KIND, TQ, TP, GATED, EPI, 128, 128, 2, 2, 2>(a, p, 2, st);
    case G128X128: return launch_gemm<KIND, TQ, TP, GATED, EPI, 128, 128, 4, 2, 4>(a, p, 1, st);
    case G64X128X2: return launch_gemm<KIND, TQ, TP, GATED, EPI, 64, 128, 2, 2, 3>(a, p, 2, st);
    case G64X64X3:
      if constexpr (!GATED) return launch_gemm<KIND, TQ, TP, GATED, EPI, 64, 64, 2, 2, 3>(a, p, 3, st);
      break;
  }
  return set_error(MI355MOE_ERR_UNSUPPORTED, "gemm: no such tile");
}

}  // namespace mi355
