// The products of a backward pass (product.h) on operands that direct copies to LDS can
// fetch: BI x BJ tiles, stages of 64 r.
//
// LDS.  An operand that lies along r (q of dx) is staged as linear_tile.hip's are: 128
// bytes of each row, 16-byte chunk c of row i at slot c ^ swz(i).  One that lies across r
// (p, and the transposed q) is staged as it is, 64 rows of the tile's columns; the
// transposing LDS read gives each lane 4 r of its column, two reads a fragment.  A group of
// 16 lanes reads 32 bytes of 4 rows, 32 lanes 64 bytes of them, so chunks of consecutive
// rows are moved by 64 bytes (cross_swz): the 4 rows then cover all 64 banks once.
//
// 32x32x16 MFMAs, p's columns as the A operand, so that a lane's sums are consecutive
// columns of one row of out; four steps of 16 r per stage, the next step's fragments read
// while this one's MFMAs run; the barrier that publishes the next stage sits before the
// last step.  Rows and columns past the edges repeat the last ones and are not stored;
// the last stage's r past R are cleared in LDS.
#include "product.h"
#include "tile.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int BR = 64;           // r of a stage
constexpr int SB = 2 * BR;       // bytes of a stage in a row along r
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }
// staged across r: chunk c of row r is at slot c ^ cross_swz<chunks of a row>(r)
template <int CH>
__device__ __forceinline__ int cross_swz(int r) {
  return CH >= 16 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}

template <bool F16, bool TQ, int BI, int BJ, int WI, int WJ, int NSTAGE>
__global__ __launch_bounds__(64 * WI * WJ) void product_tile_kernel(const Product a, float* part,
                                                                     int tiles_i, int tiles_j,
                                                                     int splits, int stages_per_split) {
  constexpr int WAVES = WI * WJ, THREADS = 64 * WAVES;
  constexpr int MT = BI / WI / 32, NT = BJ / WJ / 32;
  static_assert(MT >= 1 && NT >= 1, "wave tile");
  constexpr int STAGE = (BI + BJ) * SB;
  constexpr int PCH = BJ / 8, QCH = TQ ? BI / 8 : SB / 16;    // 16-byte chunks of a staged row
  constexpr int PRC = 64 / PCH, QRC = 64 / QCH;               // rows of a 1 KB copy
  constexpr int QQ = BI / 8 / WAVES, PQ = BJ / 8 / WAVES, ND = QQ + PQ;  // copies per wave and stage
  static_assert(QQ * 8 * WAVES == BI && PQ * 8 * WAVES == BJ, "copies");
  constexpr int EM = 64, EP = BJ + 4;
  constexpr int LDS = NSTAGE * STAGE > EM * EP * 4 ? NSTAGE * STAGE : EM * EP * 4;
  static_assert(LDS <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave / WJ, wj = wave % WJ;

  // XCD i takes a contiguous range of tiles, in bands of 8 tiles of q (as linear_tile.hip)
  const int total = tiles_i * tiles_j * splits;
  const int per = (total + 7) / 8;
  const int bid = static_cast<int>(blockIdx.x);
  int t = (bid & 7) * per + (bid >> 3);
  if ((bid >> 3) >= per || t >= total) return;  // uniform
  const int split = t / (tiles_i * tiles_j);
  t %= tiles_i * tiles_j;
  constexpr int BAND = 8;
  const int band = t / (BAND * tiles_j);
  const int bi = tiles_i - band * BAND < BAND ? tiles_i - band * BAND : BAND;
  t -= band * BAND * tiles_j;
  const int64_t i0 = static_cast<int64_t>(band * BAND + t % bi) * BI;
  const int64_t j0 = static_cast<int64_t>(t / bi) * BJ;

  const int nk_all = static_cast<int>((a.R + BR - 1) / BR);
  const int k0 = split * stages_per_split;
  const int nk = nk_all - k0 < stages_per_split ? nk_all - k0 : stages_per_split;
  const int tail = k0 + nk == nk_all ? static_cast<int>(a.R % BR) : 0;  // r of the last stage, 0: all

  // copy q of this wave: block wave QQ + q of the staged q, then wave PQ + (q - QQ) of p;
  // offsets from the tile's first row (along r) or from the stage's first row (across)
  const uint64_t qbase = uniform_ptr(static_cast<const uint8_t*>(a.q) + (TQ ? i0 * 2 : i0 * a.ldq * 2));
  const uint64_t pbase = uniform_ptr(static_cast<const uint8_t*>(a.p) + j0 * 2);
  const uint64_t qstep = TQ ? static_cast<uint64_t>(a.ldq) * (2 * BR) : SB;
  const uint64_t pstep = static_cast<uint64_t>(a.ldp) * (2 * BR);
  // (q across r: its rows are readable to a multiple of 8 columns)
  const int qlast = static_cast<int>(TQ ? ((a.I + 7) / 8 - i0 / 8 < QCH ? (a.I + 7) / 8 - i0 / 8 : QCH) - 1 : 0);
  const int plast = static_cast<int>((a.J / 8 - j0 / 8 < PCH ? a.J / 8 - j0 / 8 : PCH) - 1);
  auto row_of = [=](int q) __attribute__((always_inline)) {
    return q < QQ ? (wave * QQ + q) * QRC + lane / QCH : (wave * PQ + q - QQ) * PRC + lane / PCH;
  };
  uint32_t voff[ND];
#pragma unroll
  for (int q = 0; q < ND; ++q) {
    const int r = row_of(q);
    if (q < QQ && !TQ) {
      const int64_t last = a.I - 1 - i0;
      voff[q] = static_cast<uint32_t>((r < last ? r : last) * a.ldq * 2 + (((lane % QCH) ^ swz(r)) << 4));
    } else {
      const int c = q < QQ ? (lane % QCH) ^ cross_swz<QCH>(r) : (lane % PCH) ^ cross_swz<PCH>(r);
      const int last = q < QQ ? qlast : plast;
      voff[q] = static_cast<uint32_t>(r * (q < QQ ? a.ldq : a.ldp) * 2 + ((c < last ? c : last) << 4));
    }
  }
  const uint32_t ring = lds_off(lds);
  // copy Q into the slot at LDS offset `slot`; past: the stage holds `tail` r, rows behind
  // them repeat the last, chunks behind them the stage's first
  auto copy = [=](auto qc, uint64_t qoff, uint64_t poff, uint32_t slot, bool past)
      __attribute__((always_inline)) {
    constexpr int Q = decltype(qc)::value;
    constexpr bool X = Q < QQ;
    uint32_t v = voff[Q];
    if (past) {  // uniform
      const int r = row_of(Q);
      if (X && !TQ) {
        const int cb = ((lane % QCH) ^ swz(r)) << 4;
        if (cb >= 2 * tail) v -= cb;
      } else if (r >= tail) {
        v -= static_cast<uint32_t>((r - (tail - 1)) * (X ? a.ldq : a.ldp) * 2);
      }
    }
    if constexpr (X) dma16<Q * 1024>(v, qbase + qoff, slot + wave * (QQ * 1024));
    else dma16<BI * SB + (Q - QQ) * 1024>(v, pbase + poff, slot + wave * (PQ * 1024));
  };
  auto issue = [=](int kt) __attribute__((always_inline)) {
    const uint32_t slot = ring + (kt % NSTAGE) * STAGE;
    const bool past = tail != 0 && kt == nk - 1;
    for_each<ND>([&](auto q) __attribute__((always_inline)) {
      copy(q, static_cast<uint64_t>(k0 + kt) * qstep, static_cast<uint64_t>(k0 + kt) * pstep, slot, past);
    });
  };
  // the last stage's r behind `tail` (q along r: to its multiple of 8, where zeros follow)
  auto clear_tail = [=](int kt) __attribute__((always_inline)) {
    uint8_t* S = lds + (kt % NSTAGE) * STAGE;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    if constexpr (TQ) {
      for (int i = tail * QCH + tid; i < BR * QCH; i += THREADS) reinterpret_cast<uint4*>(S)[i] = zero;
    } else {
      for (int i = tid; i < BI * QCH; i += THREADS) {
        const int r = i / QCH, c = i % QCH;
        if (8 * c >= tail) *reinterpret_cast<uint4*>(S + r * SB + ((c ^ swz(r)) << 4)) = zero;
      }
    }
    for (int i = tail * PCH + tid; i < BR * PCH; i += THREADS)
      reinterpret_cast<uint4*>(S + BI * SB)[i] = zero;
    lds_barrier();
  };

  for (int s = 0; s < NSTAGE && s < nk; ++s) issue(s);
  if (nk >= NSTAGE) wait_vm<ND * (NSTAGE - 1)>();
  else wait_vm<0>();
  __builtin_amdgcn_s_barrier();
  if (tail && nk == 1) clear_tail(0);
  // publishes stage kt + 1; every wave has read stage kt then
  auto advance = [=](int kt) __attribute__((always_inline)) {
    if (kt + 1 >= nk) return;
    if (kt + NSTAGE <= nk) wait_vm<ND * (NSTAGE - 2)>();
    else wait_vm<0>();
    lds_barrier();
    if (tail && kt + 2 == nk) clear_tail(kt + 1);
  };

  f32x16 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // Where this lane reads fragment n of an operand: across r, row 8 h + t / 4 (then + 4) of a
  // K step, 4 columns from 16 (g & 1) + 4 (t & 3) of the fragment's 32; along r, chunk h of
  // row l32.
  const int g = lane >> 4, tl = lane & 15, h = lane >> 5, l32 = lane & 31;
  auto cross_at = [=](auto ch, int col) __attribute__((always_inline)) {
    constexpr int CH = decltype(ch)::value;
    const int r = 8 * h + (tl >> 2);
    return r * (CH * 16) + (((col / 8) ^ cross_swz<CH>(r)) << 4) +
           ((2 * (g & 1) + ((tl & 3) >> 1)) << 4) + 8 * (tl & 1);
  };
  int pat[NT], qat[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    pat[i] = BI * SB + cross_at(std::integral_constant<int, PCH>{}, wj * (BJ / WJ) + 32 * i);
#pragma unroll
  for (int j = 0; j < MT; ++j)
    qat[j] = TQ ? cross_at(std::integral_constant<int, TQ ? QCH : 8>{}, wi * (BI / WI) + 32 * j)
                : (wi * (BI / WI) + 32 * j + l32) * SB;
  const int sw = swz(l32);

  constexpr int KS = BR / 16;
  struct Frag {
    uint4 q[MT], p[NT];
  };
  Frag f[2];
  constexpr int NF = MT + NT;
  auto cross8 = [&](const uint8_t* s, int row) __attribute__((always_inline)) {
    const uint2 lo = lds_column4(s), hi = lds_column4(s + 4 * row);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  auto read = [&](Frag& o, const uint8_t* S, int ks, int e) __attribute__((always_inline)) {
    if (e == 0 || e > MT) {
      const int i = e == 0 ? 0 : e - MT;
      o.p[i] = cross8(S + pat[i] + ks * (16 * PCH * 16), PCH * 16);
    } else if (TQ) {
      o.q[e - 1] = cross8(S + qat[e - 1] + ks * (16 * QCH * 16), QCH * 16);
    } else {
      o.q[e - 1] = lds16(S + qat[e - 1] + (((2 * ks + h) ^ sw) << 4));
    }
  };
  constexpr int NM = NT * MT, RPM = (NF + NM - 1) / NM, CPM = (ND + NM - 1) / NM;
  auto step = [&](auto last_c, bool dma, const Frag& c, Frag& next, const uint8_t* Sn, int kn,
                  uint64_t qoff, uint64_t poff, uint32_t slot) __attribute__((always_inline)) {
    for_each<NM>([&](auto tc) __attribute__((always_inline)) {
      constexpr int m = decltype(tc)::value, i = m / MT, j = m % MT;
      acc[i][j] = mfma16_32x32x16<F16>(c.p[i], c.q[j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = m * RPM; e < (m + 1) * RPM && e < NF; ++e) read(next, Sn, kn, e);
      if constexpr (decltype(last_c)::value && m * CPM < ND) {
        if (dma) {
          for_each<CPM>([&](auto cc) __attribute__((always_inline)) {
            constexpr int Q = m * CPM + decltype(cc)::value;
            if constexpr (Q < ND) copy(std::integral_constant<int, Q>{}, qoff, poff, slot, false);
          });
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
#pragma unroll
  for (int e = 0; e < NF; ++e) read(f[0], lds, 0, e);
  const int nfull = tail ? nk - 1 : nk;
  uint64_t qoff = static_cast<uint64_t>(k0 + NSTAGE) * qstep, poff = static_cast<uint64_t>(k0 + NSTAGE) * pstep;
  int slot = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const uint8_t* S = lds + slot * STAGE;
    const int nslot = slot + 1 == NSTAGE ? 0 : slot + 1;
    const uint8_t* Sn = lds + nslot * STAGE;
#pragma unroll
    for (int ks = 0; ks + 1 < KS; ++ks)
      step(std::false_type{}, false, f[ks & 1], f[(ks + 1) & 1], S, ks + 1, 0, 0, 0);
    advance(kt);
    if (tail && kt + NSTAGE == nk - 1) issue(kt + NSTAGE);
    // after the last stage this reads a stale slot, unused
    step(std::true_type{}, kt + NSTAGE < nfull, f[(KS - 1) & 1], f[0], Sn, 0, qoff, poff,
         ring + slot * STAGE);
    qoff += qstep;
    poff += pstep;
    slot = nslot;
  }

  // ---- epilogue: 64 rows at a time through LDS to threads that own 8 columns
  float* ep = reinterpret_cast<float*>(lds);
  constexpr int RUNS = BJ / 8, ITEMS = EM * RUNS / THREADS;
  static_assert(ITEMS * THREADS == EM * RUNS, "epilogue");
  const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * 2)) & 15) == 0;
#pragma unroll 1
  for (int s = 0; s < BI / EM; ++s) {
    const int64_t is = i0 + s * EM;
    if (is >= a.I) break;  // uniform
    lds_barrier();  // the ring, or the pass before, is read
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int row0 = wi * (BI / WI) + 32 * j - s * EM;
      if (row0 < 0 || row0 >= EM) continue;  // uniform
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<f32x4*>(ep + (row0 + l32) * EP + wj * (BJ / WJ) + 32 * i + 8 * k + 4 * h) =
              f32x4{acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]};
    }
    lds_barrier();
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      const int idx = e * THREADS + tid;
      const int row = idx / RUNS, c = (idx % RUNS) * 8;
      const int64_t i = is + row, j = j0 + c;
      if (i >= a.I || j >= a.J) continue;  // (J is whole runs)
      const f32x4 lo = *reinterpret_cast<const f32x4*>(ep + row * EP + c);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(ep + row * EP + c + 4);
      if (splits > 1) {
        f32x4* o = reinterpret_cast<f32x4*>(part + (static_cast<int64_t>(split) * a.I + i) * a.J + j);
        o[0] = lo;
        o[1] = hi;
      } else {
        uint16_t* o = static_cast<uint16_t*>(a.out) + i * a.ldo + j;
        const uint4 w = make_uint4(pack16x2<F16>(lo[0], lo[1]), pack16x2<F16>(lo[2], lo[3]),
                                   pack16x2<F16>(hi[0], hi[1]), pack16x2<F16>(hi[2], hi[3]));
        if (vec) {
          *reinterpret_cast<uint4*>(o) = w;
        } else {
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = static_cast<uint16_t>(u[k >> 1] >> (16 * (k & 1)));
        }
      }
    }
  }
}

// The tiles that calls choose from, and the time of one stage on every CU at once.
enum Shape { T256X256, T128X128X2, T128X128, T64X128, T64X64 };
struct Tile {
  Shape shape;
  int bi, bj, per_cu;
  float us;
};
constexpr Tile kTiles[] = {{T256X256, 256, 256, 1, 1.95f}, {T128X128X2, 128, 128, 2, 1.25f},
                           {T128X128, 128, 128, 1, 0.72f}, {T64X128, 64, 128, 1, 0.46f},
                           {T64X64, 64, 64, 1, 0.33f}};
constexpr int kMaxSplits = 16;
constexpr int kMaxSplitTiles = 1 << 16;

struct Plan {
  Shape shape;
  int splits, per;
};
// The tile and the split of R with the least estimated time (as linear_tile.hip's): rounds of
// the grid over the CUs, each its stages and 3 us around them, and for a split the partial
// sums written and read at 3.5 TB/s and a second launch.
Plan plan(const Product& p) {
  const int nk = static_cast<int>(cdiv(p.R, BR));
  Plan best{};
  double best_us = -1;
  for (const Tile& c : kTiles)
    for (int s = 1; s <= kMaxSplits; ++s) {
      const int per = static_cast<int>(cdiv(nk, s));
      if (s > 1 && (per < 4 || cdiv(nk, per) != s)) continue;
      const double tiles = static_cast<double>(cdiv(p.I, c.bi)) * cdiv(p.J, c.bj) * s;
      if (s > 1 && tiles > kMaxSplitTiles) continue;
      const double rounds = __builtin_ceil(tiles / (256.0 * c.per_cu));
      double us = rounds * (c.us * per + 3.0);
      if (s > 1) us += 4.0 + 2.0 * s * p.I * p.J * 4 / 3.5e6;
      if (best_us < 0 || us < best_us) {
        best = {c.shape, s, per};
        best_us = us;
      }
    }
  return best;
}

template <bool F16, bool TQ, int BI, int BJ, int WI, int WJ, int NSTAGE>
int launch(const Product& a, const Plan& p, float* part, hipStream_t st) {
  const int ti = static_cast<int>(cdiv(a.I, BI)), tj = static_cast<int>(cdiv(a.J, BJ));
  const dim3 grid(static_cast<unsigned>(cdiv(static_cast<int64_t>(ti) * tj * p.splits, 8) * 8));
  product_tile_kernel<F16, TQ, BI, BJ, WI, WJ, NSTAGE>
      <<<grid, dim3(64 * WI * WJ), 0, st>>>(a, part, ti, tj, p.splits, p.per);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}
template <bool F16, bool TQ>
int launch_shape(const Product& a, const Plan& p, float* part, hipStream_t st) {
  switch (p.shape) {
    case T256X256: return launch<F16, TQ, 256, 256, 2, 4, 2>(a, p, part, st);
    case T128X128X2: return launch<F16, TQ, 128, 128, 2, 2, 2>(a, p, part, st);
    case T128X128: return launch<F16, TQ, 128, 128, 2, 2, 4>(a, p, part, st);
    case T64X128: return launch<F16, TQ, 64, 128, 2, 2, 4>(a, p, part, st);
    default: return launch<F16, TQ, 64, 64, 2, 2, 8>(a, p, part, st);
  }
}

}  // namespace

bool product_tile_supported(const Product& p) {
  const int64_t lim = int64_t(1) << 32;
  auto rows16 = [](const void* b, int64_t ld) {
    return ((reinterpret_cast<uintptr_t>(b) | static_cast<uintptr_t>(ld * 2)) & 15) == 0;
  };
  return p.R > 0 && rows16(p.q, p.ldq) && rows16(p.p, p.ldp) && p.J % 8 == 0 &&
         256 * p.ldq * 2 < lim && 256 * p.ldp * 2 < lim && p.R < (int64_t(1) << 30) &&
         cdiv(p.I, 64) * cdiv(p.J, 64) < (int64_t(1) << 24);  // a grid's threads stay below 2^32
}
int product_tile_splits(const Product& p) { return plan(p).splits; }
int launch_product_tile(const Product& p, float* part, hipStream_t st) {
  const Plan n = plan(p);
  if (p.dtype == MI355MOE_F16)
    return p.transposed ? launch_shape<true, true>(p, n, part, st) : launch_shape<true, false>(p, n, part, st);
  return p.transposed ? launch_shape<false, true>(p, n, part, st) : launch_shape<false, false>(p, n, part, st);
}

}  // namespace mi355
