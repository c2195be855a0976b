// mi355moe_linear for more rows than the streaming kernels take: BM x BN tiles
// (rows of x, rows of the weight) whose K stages reach LDS by direct
// global->LDS copies.
//
// LDS.  A stage holds 128 bytes of each row of the tile, rows one after the
// other; 16-byte chunk c of row r sits at slot c ^ swz(r), so that the 16 rows
// that a quarter of a fragment read covers hit all 64 banks once.  A ring of
// NSTAGE stages; stage kt + NSTAGE is requested as soon as every wave has read
// stage kt, so NSTAGE - 1 stages are in flight.
//
// 16-bit operands: 32x32x16 MFMAs, four K steps per stage, the next step's
// fragments read while this one's MFMAs run; the barrier that publishes stage
// kt + 1 sits before the last step of stage kt, so that the matrix cores do not
// start a stage behind its reads.
// e4m3 operands: a stage is one scale block of 128; the weight's fragments of
// a stage stay in registers, x's are read one tile ahead; 16x16x128 MFMAs from
// zero, each result times x_scale * weight_scale added to the sum.  EXACT
// (float32 outputs): the fragments become bf16 and 16x16x32 MFMAs add them
// (linear.h says what the 128-long one loses).
//
// Padding.  Rows past the edges repeat the last one, their results are not
// stored; the last stage's columns past K are cleared in LDS.
//
// The tile's sums go through LDS, 64 rows of x at a time, to threads that own 8
// consecutive outputs: bias, activation, residual and stores run along rows.
#include "linear.h"
#include "tile.h"

namespace mi355 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int SB = 128;  // bytes of a row in a K stage: one e4m3 scale block, 64 16-bit values
// slot of 16-byte chunk c of row r: c ^ swz(r)
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

template <int KIND, bool GATED, bool UNI, int BM, int BN, int WM, int WN, int NSTAGE>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile_kernel(const LinArgs a, int tiles_m,
                                                                    int tiles_n, int splits,
                                                                    int stages_per_split) {
  constexpr bool FP8 = KIND >= K_FP8;
  static_assert(FP8 || UNI, "scale blocks");
  constexpr int EB = FP8 ? 1 : 2;
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  constexpr int TS = FP8 ? 16 : 32;              // MFMA tile side
  constexpr int MT = BM / WM / TS, NT = BN / WN / TS;
  static_assert(MT >= 1 && NT >= (GATED ? 2 : 1) && (!GATED || NT % 2 == 0), "wave tile");
  constexpr int BNO = GATED ? BN / 2 : BN;       // output columns
  constexpr int CH = SB / 16;                    // 16-byte chunks of a row
  constexpr int RPB = 1024 / SB;                 // rows of a 1 KB copy
  constexpr int SCALES = FP8 ? 4 * (BM + BN) : 0;
  constexpr int STAGE = (BM + BN) * SB + SCALES;
  // copies per wave and stage: XQ of x, WQ of each region of the weight
  constexpr int WREG = GATED ? 2 : 1;
  constexpr int XQ = BM / RPB / WAVES, WQ = BN / WREG / RPB / WAVES, PER = XQ + WREG * WQ;
  static_assert(XQ * RPB * WAVES == BM && WQ * RPB * WAVES * WREG == BN, "copies");
  constexpr int SC = FP8 ? (BM + BN) / 64 : 0;   // scale copies of a stage
  constexpr int SPER = (SC + WAVES - 1) / WAVES;
  constexpr int ND = PER + SPER;
  constexpr int EM = BM % 64 ? 32 : 64;          // rows of x per pass of the epilogue
  constexpr int EP = BN + 4;                     // its pitch in floats
  constexpr int LDS = NSTAGE * STAGE > EM * EP * 4 ? NSTAGE * STAGE : EM * EP * 4;
  static_assert(LDS <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
  static_assert(STAGE % 1024 == 0 || FP8, "stage alignment");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Workgroups are dealt round-robin to the 8 XCDs: XCD i takes a contiguous
  // range of tiles, ordered in bands of 8 tiles of x, so that the tiles that
  // run together on an XCD share rows of both operands in its L2.
  const int total = tiles_m * tiles_n * splits;
  const int per = (total + 7) / 8;
  const int bid = static_cast<int>(blockIdx.x);
  int t = (bid & 7) * per + (bid >> 3);
  if ((bid >> 3) >= per || t >= total) return;  // uniform
  const int split = t / (tiles_m * tiles_n);
  t %= tiles_m * tiles_n;
  constexpr int BAND = 8;
  const int band = t / (BAND * tiles_n);
  const int bm = tiles_m - band * BAND < BAND ? tiles_m - band * BAND : BAND;
  t -= band * BAND * tiles_n;
  const int64_t m0 = static_cast<int64_t>(band * BAND + t % bm) * BM;
  const int64_t n0 = static_cast<int64_t>(t / bm) * BNO;

  const int kbytes = static_cast<int>(a.K) * EB;
  const int nk_all = (kbytes + SB - 1) / SB;
  const int k0 = split * stages_per_split;       // first stage of this split
  const int nk = nk_all - k0 < stages_per_split ? nk_all - k0 : stages_per_split;
  // bytes of the last stage, 0: all (e4m3: K is whole blocks)
  const int tail = !FP8 && k0 + nk == nk_all ? kbytes % SB : 0;

  // Copies of this wave: copy q is block wave XQ + q of x's RPB-row blocks, or
  // block wave WQ + (q - XQ) % WQ of weight region (q - XQ) / WQ.  Offsets are
  // relative to the tile's first row of the region.
  const uint64_t xbase = uniform_ptr(static_cast<const uint8_t*>(a.x) + m0 * a.ldx * EB);
  const uint64_t wbase = uniform_ptr(static_cast<const uint8_t*>(a.weight) + n0 * a.ldw * EB);
  const uint64_t ubase = GATED ? uniform64(wbase + a.N * a.ldw * EB) : wbase;
  uint32_t voff[PER];
  const int cslot = lane % CH, rsub = lane / CH;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    // (the regions start at multiples of 16 rows, so a row's swizzle is its own)
    const int r = (q < XQ ? wave * XQ + q : wave * WQ + (q - XQ) % WQ) * RPB + rsub;
    const int cb = (cslot ^ swz(r)) << 4;
    const int64_t last = q < XQ ? a.M - 1 - m0 : a.N - 1 - n0;
    voff[q] = static_cast<uint32_t>((r < last ? r : last) * (q < XQ ? a.ldx : a.ldw) * EB + cb);
  }
  // e4m3: scale copies of 64 rows each, x's first
  uint32_t soff[SPER > 0 ? SPER : 1];
  uint64_t ssb[SPER > 0 ? SPER : 1];
  uint32_t sstep[SPER > 0 ? SPER : 1];
  int sblk[SPER > 0 ? SPER : 1];
  if constexpr (FP8) {
#pragma unroll
    for (int q = 0; q < SPER; ++q) {
      const int b = (SPER * wave + q) % SC;        // a surplus copy repeats one
      sblk[q] = b;
      const int r = b * 64 + lane;
      if (b < BM / 64) {
        const int64_t m = m0 + r < a.M ? r : a.M - 1 - m0;
        soff[q] = static_cast<uint32_t>(m * a.x_scale_row * 4);
        ssb[q] = uniform_ptr(a.x_scale + m0 * a.x_scale_row);
        sstep[q] = static_cast<uint32_t>(a.x_scale_blk * 4);
      } else {
        const int rr = r - BM;
        const bool up = GATED && rr >= BNO;
        int64_t n = n0 + rr - (up ? BNO : 0);
        n = (n < a.N ? n : a.N - 1) + (up ? a.N : 0);
        soff[q] = static_cast<uint32_t>((n / 128) * a.weight_scale_row * 4);
        ssb[q] = uniform_ptr(a.weight_scale);
        sstep[q] = static_cast<uint32_t>(a.weight_scale_blk * 4);
      }
    }
  }
  const uint32_t ring = lds_off(lds);
  // copy Q of a stage whose bytes start `koff` into the rows, into the slot at
  // LDS offset `slot`; TAIL: columns past K (chunks from byte `tail` on) read the
  // stage's first chunk and are cleared later
  auto copy = [=](auto qc, uint64_t koff, uint32_t slot, bool past) __attribute__((always_inline)) {
    constexpr int Q = decltype(qc)::value;
    constexpr bool X = Q < XQ;
    constexpr int REG = X ? 0 : (Q - XQ) / WQ;
    uint32_t v = voff[Q];
    if (past) {  // uniform
      const int r = (X ? wave * XQ + Q : wave * WQ + (Q - XQ) % WQ) * RPB + rsub;
      const int cb = (cslot ^ swz(r)) << 4;
      if (cb >= tail) v -= cb;
    }
    if constexpr (X) dma16<Q * 1024>(v, xbase + koff, slot + wave * (XQ * 1024));
    else
      dma16<BM * SB + REG * (BN / 2) * SB + ((Q - XQ) % WQ) * 1024>(
          v, (REG ? ubase : wbase) + koff, slot + wave * (WQ * 1024));
  };
  auto copy_scale = [=](int e, int kt, uint32_t slot) __attribute__((always_inline)) {
    dma4(soff[e], uniform64(ssb[e] + static_cast<uint64_t>(k0 + kt) * sstep[e]),
         __builtin_amdgcn_readfirstlane(slot + (BM + BN) * SB + sblk[e] * 256));
  };
  // a whole stage
  auto issue = [=](int kt) __attribute__((always_inline)) {
    const uint32_t slot = ring + (kt % NSTAGE) * STAGE;
    const uint64_t koff = static_cast<uint64_t>(k0 + kt) * SB;
    const bool past = tail != 0 && kt == nk - 1;
    for_each<PER>([&](auto q) __attribute__((always_inline)) { copy(q, koff, slot, past); });
    if constexpr (FP8) {
#pragma unroll
      for (int e = 0; e < SPER; ++e) copy_scale(e, kt, slot);
    }
  };
  // the last stage's columns past K
  auto clear_tail = [=](int kt) __attribute__((always_inline)) {
    uint8_t* S = lds + (kt % NSTAGE) * STAGE;
    for (int i = tid; i < (BM + BN) * CH; i += THREADS) {
      const int r = i / CH, c = i % CH;
      if ((c << 4) >= tail)
        *reinterpret_cast<uint4*>(S + r * SB + ((c ^ swz(r)) << 4)) = make_uint4(0, 0, 0, 0);
    }
    lds_barrier();
  };

  for (int s = 0; s < NSTAGE && s < nk; ++s) issue(s);
  if (nk >= NSTAGE) wait_vm<ND * (NSTAGE - 1)>();
  else wait_vm<0>();

  __builtin_amdgcn_s_barrier();
  if (tail && nk == 1) clear_tail(0);

  // publishes stage kt + 1; every wave has read stage kt then, so that stage kt +
  // NSTAGE may go to its slot
  auto advance = [=](int kt) __attribute__((always_inline)) {
    if (kt + 1 >= nk) return;
    if (kt + NSTAGE <= nk) wait_vm<ND * (NSTAGE - 2)>();
    else wait_vm<0>();
    lds_barrier();
    if (tail && kt + 2 == nk) clear_tail(kt + 1);
  };

  using Acc = std::conditional_t<FP8, f32x4, f32x16>;
  constexpr int AR = FP8 ? 4 : 16;
  Acc acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int r = 0; r < AR; ++r) acc[i][j][r] = 0.f;

  // weight tile i's first row in the stage: gated waves take the same columns
  // of both halves
  auto wrow = [&](int i) __attribute__((always_inline)) {
    if constexpr (GATED)
      return i < NT / 2 ? wn * (BNO / WN) + TS * i : BNO + wn * (BNO / WN) + TS * (i - NT / 2);
    else
      return wn * (BN / WN) + TS * i;
  };

  if constexpr (!FP8) {
    constexpr int KS = SB / 32;  // K steps of 16 per stage
    const int l32 = lane & 31, h = lane >> 5;
    struct Frag {
      uint4 x[MT], w[NT];
    };
    Frag f[2];
    const int sw = swz(l32);  // rows l32 + 32 i share it
    // fragment e of a K step, in the order that the MFMAs want them
    constexpr int NF = MT + NT;
    auto read = [&](Frag& g, const uint8_t* S, int ks, int e) __attribute__((always_inline)) {
      const int c = ((2 * ks + h) ^ sw) << 4;
      if (e == 0 || e > MT) {
        const int i = e == 0 ? 0 : e - MT;
        g.w[i] = lds16(S + (BM + wrow(i) + l32) * SB + c);
      } else {
        g.x[e - 1] = lds16(S + (wm * (BM / WM) + 32 * (e - 1) + l32) * SB + c);
      }
    };
    // One K step: its MFMAs, between them the reads of the next step's fragments
    // (kn of stage Sn) and, with `dma`, the copies of a stage; the order is kept.
    // (`dma`, uniform, guards the copies alone: two versions of the step would
    // have the compiler copy every accumulator where they join.)
    constexpr int NM = NT * MT, RPM = (NF + NM - 1) / NM, CPM = (PER + NM - 1) / NM;
    auto step = [&](auto last_c, bool dma, const Frag& g, Frag& next, const uint8_t* Sn, int kn,
                    uint64_t koff, uint32_t slot) __attribute__((always_inline)) {
      for_each<NM>([&](auto tc) __attribute__((always_inline)) {
        constexpr int t = decltype(tc)::value, i = t / MT, j = t % MT;
        acc[i][j] = mfma16_32x32x16<KIND == K_F16>(g.w[i], g.x[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = t * RPM; e < (t + 1) * RPM && e < NF; ++e) read(next, Sn, kn, e);
        if constexpr (decltype(last_c)::value && t * CPM < PER) {
          if (dma) {
            for_each<CPM>([&](auto c) __attribute__((always_inline)) {
              constexpr int Q = t * CPM + decltype(c)::value;
              if constexpr (Q < PER) copy(std::integral_constant<int, Q>{}, koff, slot, false);
            });
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    };
#pragma unroll
    for (int e = 0; e < NF; ++e) read(f[0], lds, 0, e);
    // stages [NSTAGE, nfull) are requested between MFMAs, a partial last one at once
    const int nfull = tail ? nk - 1 : nk;
    uint64_t koff = static_cast<uint64_t>(k0 + NSTAGE) * SB;
    int slot = 0;
    for (int kt = 0; kt < nk; ++kt) {
      const uint8_t* S = lds + slot * STAGE;
      const int nslot = slot + 1 == NSTAGE ? 0 : slot + 1;
      const uint8_t* Sn = lds + nslot * STAGE;
#pragma unroll
      for (int ks = 0; ks + 1 < KS; ++ks)
        step(std::false_type{}, false, f[ks & 1], f[(ks + 1) & 1], S, ks + 1, 0, 0);
      advance(kt);
      if (tail && kt + NSTAGE == nk - 1) issue(kt + NSTAGE);
      // after the last stage this reads a stale slot, unused
      step(std::true_type{}, kt + NSTAGE < nfull, f[(KS - 1) & 1], f[0], Sn, 0, koff,
           ring + slot * STAGE);
      koff += SB;
      slot = nslot;
    }
  } else {
    const int l16 = lane & 15, q = lane >> 4;
    const int sw16 = swz(l16);
    // operand bytes 0-15 from chunk q, 16-31 from chunk 4 + q: both operands the
    // same, so the order within the block does not matter
    const int c0 = (q ^ sw16) << 4, c1 = ((4 + q) ^ sw16) << 4;
    for (int kt = 0; kt < nk; ++kt) {
      const uint8_t* S = lds + (kt % NSTAGE) * STAGE;
      const float* sx = reinterpret_cast<const float*>(S + (BM + BN) * SB);
      const float* sw = sx + BM;
      // copies of the stage after next into the slot that the last one left
      const int kn = kt + NSTAGE - 1;
      const bool dma = kt > 0 && kn < nk;
      const uint32_t nslot = ring + (kn % NSTAGE) * STAGE;
      const uint64_t koff = static_cast<uint64_t>(k0 + kn) * SB;
      if constexpr (KIND == K_FP8) {
        auto frag = [&](int row) __attribute__((always_inline)) {
          const uint8_t* p = S + (row + l16) * SB;
          const uint4 u0 = lds16(p + c0), u1 = lds16(p + c1);
          return i32x8{(int)u0.x, (int)u0.y, (int)u0.z, (int)u0.w,
                       (int)u1.x, (int)u1.y, (int)u1.z, (int)u1.w};
        };
        i32x8 w[NT], x[2];
        float xs[3];  // of x tiles j - 1, j, j + 1
        // UNI: the 16 weight rows of a tile share one scale block
        using Ws = std::conditional_t<UNI, float, f32x4>;
        Ws ws[NT];
        x[0] = frag(wm * (BM / WM));
        xs[0] = sx[wm * (BM / WM) + l16];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          w[i] = frag(BM + wrow(i));
          if constexpr (UNI) ws[i] = sw[wrow(i)];
          else ws[i] = *reinterpret_cast<const f32x4*>(sw + wrow(i) + 4 * q);
        }
        // a result is scaled and added while the next MFMA runs
        f32x4 d[2];
        auto add = [&](auto ec) __attribute__((always_inline)) {
          constexpr int e = decltype(ec)::value, i = e % NT, j = e / NT;
          if constexpr (UNI) {
            const float f = xs[j % 3] * ws[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] += d[e & 1][r] * f;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] += d[e & 1][r] * (xs[j % 3] * ws[i][r]);
          }
        };
        constexpr int CPM = (ND + MT * NT - 1) / (MT * NT);  // copies behind an MFMA
        for_each<MT>([&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value;
          if constexpr (j + 1 < MT) {
            const int row = wm * (BM / WM) + 16 * (j + 1);
            x[(j + 1) & 1] = frag(row);
            xs[(j + 1) % 3] = sx[row + l16];
          }
          __builtin_amdgcn_sched_barrier(0);
          for_each<NT>([&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value;
            constexpr int Q = j * NT + i;
            d[Q & 1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                w[i], x[j & 1], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 127, 0, 127);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (Q > 0) add(std::integral_constant<int, Q - 1>{});
            if constexpr (Q * CPM < ND) {
              if (dma) {
                for_each<CPM>([&](auto cc) __attribute__((always_inline)) {
                  constexpr int C = Q * CPM + decltype(cc)::value;
                  if constexpr (C < PER) copy(std::integral_constant<int, C>{}, koff, nslot, false);
                  else if constexpr (C < ND) copy_scale(C - PER, kn, nslot);
                });
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          });
        });
        add(std::integral_constant<int, MT * NT - 1>{});
      } else {
        if (dma) issue(kn);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint8_t* p = S + (BM + wrow(i) + l16) * SB;
          const uint4 u0 = lds16(p + c0), u1 = lds16(p + c1);
          const uint4 w[4] = {fp8x8_to16<false, false>(make_uint2(u0.x, u0.y)),
                              fp8x8_to16<false, false>(make_uint2(u0.z, u0.w)),
                              fp8x8_to16<false, false>(make_uint2(u1.x, u1.y)),
                              fp8x8_to16<false, false>(make_uint2(u1.z, u1.w))};
          const f32x4 ws = *reinterpret_cast<const f32x4*>(sw + wrow(i) + 4 * q);
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const int row = wm * (BM / WM) + 16 * j + l16;
            const uint8_t* px = S + row * SB;
            const uint4 v0 = lds16(px + c0), v1 = lds16(px + c1);
            f32x4 d = {0.f, 0.f, 0.f, 0.f};
            d = mfma16_16x16x32<false>(w[0], fp8x8_to16<false, false>(make_uint2(v0.x, v0.y)), d);
            d = mfma16_16x16x32<false>(w[1], fp8x8_to16<false, false>(make_uint2(v0.z, v0.w)), d);
            d = mfma16_16x16x32<false>(w[2], fp8x8_to16<false, false>(make_uint2(v1.x, v1.y)), d);
            d = mfma16_16x16x32<false>(w[3], fp8x8_to16<false, false>(make_uint2(v1.z, v1.w)), d);
            const float xs = sx[row];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] += d[r] * (xs * ws[r]);
          }
        }
      }
      advance(kt);
    }
  }

  // ---- epilogue
  float* ep = reinterpret_cast<float*>(lds);
  LinArgs o = a;
  if (splits > 1) o.out = static_cast<float*>(a.out) + static_cast<int64_t>(split) * a.M * a.N;
  const int osize = o.out_dtype == MI355MOE_F32 ? 4 : 2;
  const bool vec = ((reinterpret_cast<uintptr_t>(o.out) | static_cast<uintptr_t>(o.ldo * osize)) & 15) == 0;
  // outputs of a pass: ITEMS runs of 8 columns per thread
  constexpr int RUNS = BNO / 8, ITEMS = EM * RUNS / THREADS;
  static_assert(ITEMS * THREADS == EM * RUNS, "epilogue");
  const bool early = o.residual && o.residual_dtype != MI355MOE_F32 && n0 + BNO <= a.N &&
                     ((reinterpret_cast<uintptr_t>(o.residual) | static_cast<uintptr_t>(o.ldr * 2)) & 15) == 0;
#pragma unroll 1
  for (int p = 0; p < BM / EM; ++p) {
    const int64_t mp = m0 + p * EM;
    if (mp >= a.M) break;  // uniform
    // the residual's loads are on their way while the sums go through LDS
    uint4 res[ITEMS];
    if (early) {
#pragma unroll
      for (int e = 0; e < ITEMS; ++e) {
        const int idx = e * THREADS + tid;
        int64_t m = mp + idx / RUNS;
        m = m < a.M ? m : a.M - 1;
        res[e] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(o.residual) + m * o.ldr +
                                                 n0 + (idx % RUNS) * 8);
      }
    }
    lds_barrier();  // the ring, or the pass before, is read
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int row0 = wm * (BM / WM) + TS * j - p * EM;
      if (row0 < 0 || row0 >= EM) continue;  // uniform
      const int row = row0 + (FP8 ? lane & 15 : lane & 31);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < AR / 4; ++g) {
          const int col = wrow(i) + (FP8 ? 4 * (lane >> 4) : 8 * g + 4 * (lane >> 5));
          *reinterpret_cast<f32x4*>(ep + row * EP + col) =
              f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
    }
    lds_barrier();
#pragma unroll
    for (int e = 0; e < ITEMS; ++e) {
      const int idx = e * THREADS + tid;
      const int row = idx / RUNS, c = (idx % RUNS) * 8;
      const int64_t m = mp + row, n = n0 + c;
      if (m >= a.M || n >= a.N) continue;
      const float* z = ep + row * EP + c;
      lin_store8(o, m, n, z, z + (GATED ? BNO : 0), vec, early, res[e]);
    }
  }
}

// The tiles that calls choose from.  us: time of one stage (128 bytes of K) on
// every CU at once; per_cu: workgroups of the tile that a CU holds; gated: takes
// both halves of a gated weight (a split product needs no gates; 16-bit 64 x 64
// with two waves of 32 x 64 gained nothing there, 200 x 2048 x 1536 13.4 -> 14.9).
enum Shape { T256X256, T128X256, T128X128X2, T128X128, T96X128, T64X128, T64X64 };
struct Tile {
  Shape shape;
  int bm, bn, per_cu;
  bool gated;
  float us;
};
// (Sizes: rows x K x weight rows, both halves of a gated weight counted.)
// 16-bit.  256 x 256: 8 waves of 128 x 64 and two stages (four of 64 bytes: 5 %
// slower; 4 waves of 128 x 128: alike); 26 (gated) and 70 registers are spilled, once
// behind the K loop, for the epilogue.  Two workgroups of 128 x 128 per CU hide
// each other's epilogues, one with four stages hides the latency where tiles are
// few.  The others fill the CUs where these leave some idle (us, K = 4096 unless
// said, best of the others after it): 128 x 256 1500 x 4096 65 / 69, 2048 x 4096
// gated 71 / 77; 96 x 128 1003 x 2880 x 2880 30.6 / 34.9, 700 x 4096 39.6 / 41.8;
// 64 x 64, eight stages, 250 x 4096 24.4 / 31.5 (64 x 128), 61 x 4096 split by 4
// 16.5 / 17.1 (64 x 128 by 8).
constexpr Tile kTiles16[] = {
    {T256X256, 256, 256, 1, true, 1.85f}, {T128X256, 128, 256, 1, true, 1.14f},
    {T128X128X2, 128, 128, 2, true, 1.16f}, {T128X128, 128, 128, 1, true, 0.66f},
    {T96X128, 96, 128, 1, false, 0.555f}, {T64X128, 64, 128, 1, true, 0.42f},
    {T64X64, 64, 64, 1, false, 0.31f}};
// e4m3.  256 x 256 leaves no registers for the scaled sums (spills: 8192 x 4096 x
// 4096 288 us, 128 x 256 210); 96 rows are no whole copies of scales.  64 x 64: 250 x
// 4096 x 4096 18.8 us (64 x 128 24.9), 61 x 2048 x 7168 12.4 (16.1), 250 x 4096 x 4096
// gated 18.2 (24.6).
constexpr Tile kTiles8[] = {
    {T128X256, 128, 256, 1, true, 1.45f}, {T128X128X2, 128, 128, 2, true, 1.73f},
    {T128X128, 128, 128, 1, true, 1.08f}, {T64X128, 64, 128, 1, true, 0.70f},
    {T64X64, 64, 64, 1, true, 0.44f}};
// e4m3 with float32 outputs (EXACT): the bf16 fragments take the registers of two
// workgroups per CU (276 to 304 of a lane's 512), so 128 x 128 with two stages runs
// alone there, and no slower than with four (1.32 and 1.39 us a stage).
constexpr Tile kTiles8Exact[] = {
    {T128X256, 128, 256, 1, true, 1.94f}, {T128X128X2, 128, 128, 1, true, 1.32f},
    {T64X128, 64, 128, 1, true, 0.85f}, {T64X64, 64, 64, 1, true, 0.59f}};
constexpr int kMaxSplits = 16;
constexpr int kMaxSplitTiles = 1 << 16;  // workgroups of a split product: far more than fill the CUs

struct Plan {
  Shape shape;
  int splits, per;  // stages per split
};

// 16 weight rows from a multiple of 16 share a scale block
bool uniform_scales(const LinArgs& a) { return !lin_gated(a.activation) || a.N % 16 == 0; }

// The tile and the split of K with the least estimated time: rounds of the
// grid over the CUs, each its stages and 3 us around them, and for a split the
// partial sums written and read at 3.5 TB/s and a second launch.
Plan plan(const LinArgs& a) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  const bool exact = fp8 && a.out_dtype == MI355MOE_F32;
  const int nk = static_cast<int>(cdiv(a.K * (fp8 ? 1 : 2), 128));
  const bool g = lin_gated(a.activation);
  const double rows = static_cast<double>(lin_rows(a));
  Plan best{};
  double best_us = -1;
  auto look = [&](const Tile& c) {
    for (int s = 1; s <= kMaxSplits; ++s) {
      const int per = static_cast<int>(cdiv(nk, s));
      if (s > 1 && (per < 4 || cdiv(nk, per) != s)) continue;
      const bool gates = g && s == 1;  // a split product: all weight rows, no gates
      if (gates && !c.gated) continue;
      const double tiles = static_cast<double>(cdiv(a.M, c.bm)) *
                           cdiv(gates ? a.N : lin_rows(a), gates ? c.bn / 2 : c.bn) * s;
      if (s > 1 && tiles > kMaxSplitTiles) continue;
      const double rounds = __builtin_ceil(tiles / (256.0 * c.per_cu));
      double us = rounds * (c.us * per + 3.0);
      if (s > 1) us += 4.0 + 2.0 * s * a.M * rows * 4 / 3.5e6;
      if (best_us < 0 || us < best_us) {
        best = {c.shape, s, per};
        best_us = us;
      }
    }
  };
  if (exact)
    for (const Tile& c : kTiles8Exact) look(c);
  else if (fp8)
    for (const Tile& c : kTiles8) look(c);
  else
    for (const Tile& c : kTiles16) look(c);
  return best;
}

template <int KIND, bool GATED, bool UNI, int BM, int BN, int WM, int WN, int NSTAGE>
int launch(const LinArgs& a, const Plan& p, hipStream_t st) {
  const int tm = static_cast<int>(cdiv(a.M, BM)), tn = static_cast<int>(cdiv(a.N, GATED ? BN / 2 : BN));
  const dim3 grid(static_cast<unsigned>(cdiv(static_cast<int64_t>(tm) * tn * p.splits, 8) * 8));
  linear_tile_kernel<KIND, GATED, UNI, BM, BN, WM, WN, NSTAGE>
      <<<grid, dim3(64 * WM * WN), 0, st>>>(a, tm, tn, p.splits, p.per);
  MI_LAUNCH_CHECK();
  return MI355MOE_OK;
}

template <int KIND, bool GATED, int BM, int BN, int WM, int WN, int NSTAGE>
int launch_uni(const LinArgs& a, const Plan& p, hipStream_t st) {
  if constexpr (KIND >= K_FP8)
    if (!uniform_scales(a)) return launch<KIND, GATED, false, BM, BN, WM, WN, NSTAGE>(a, p, st);
  return launch<KIND, GATED, true, BM, BN, WM, WN, NSTAGE>(a, p, st);
}

template <int KIND, bool GATED>
int launch_tiles(const LinArgs& a, const Plan& p, hipStream_t st) {
  if constexpr (KIND < K_FP8) {
    if (p.shape == T256X256) return launch_uni<KIND, GATED, 256, 256, 2, 4, 2>(a, p, st);
    if constexpr (!GATED)
      if (p.shape == T96X128) return launch_uni<KIND, GATED, 96, 128, 1, 4, 4>(a, p, st);
  }
  if constexpr (KIND >= K_FP8 || !GATED)
    if (p.shape == T64X64) return launch_uni<KIND, GATED, 64, 64, 2, 2, 8>(a, p, st);
  if constexpr (KIND != K_FP8_EXACT)
    if (p.shape == T128X128) return launch_uni<KIND, GATED, 128, 128, 2, 2, 4>(a, p, st);
  switch (p.shape) {
    case T128X256: return launch_uni<KIND, GATED, 128, 256, 2, 4, 3>(a, p, st);
    case T128X128X2: return launch_uni<KIND, GATED, 128, 128, 2, 2, 2>(a, p, st);
    default: return launch_uni<KIND, GATED, 64, 128, 2, 2, 4>(a, p, st);
  }
}

}  // namespace

// Operand rows that the direct copies can fetch: 16-byte aligned, whole
// 16-byte pieces, a tile's rows within 32-bit offsets of its first.
bool linear_tile_supported(const LinArgs& a) {
  const bool fp8 = a.x_dtype == MI355MOE_FP8E4M3;
  const int64_t eb = kind_bytes(kind_of(a)), lim = int64_t(1) << 32;
  auto rows16 = [&](const void* p, int64_t ld) {
    return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(ld * eb)) & 15) == 0 &&
           256 * ld * eb < lim;
  };
  if (!rows16(a.x, a.ldx) || !rows16(a.weight, a.ldw) || a.K * eb % 16) return false;
  if (fp8) {
    const int64_t blocks = cdiv(lin_rows(a), 128);
    // (block strides step a scalar base by 32 bits)
    if (256 * a.x_scale_row * 4 >= lim || a.x_scale_blk * 4 >= lim ||
        blocks * a.weight_scale_row * 4 >= lim || a.weight_scale_blk * 4 >= lim)
      return false;
  }
  // a grid's threads (256 to a tile of 64 rows of x) stay below 2^32
  return cdiv(a.M, 64) * cdiv(lin_rows(a), 64) < (int64_t(1) << 24);
}

// int8 operands and kept sums: gemm_tile.h's kernels
bool gemm_tiles(const LinArgs& a) { return a.x_dtype == MI355MOE_I8 || a.z; }

int linear_tile_splits(const LinArgs& a) {
  return gemm_tiles(a) ? linear_gemm_splits(a) : plan(a).splits;
}

int launch_linear_tile(const LinArgs& a0, const LinArgs& a, hipStream_t st) {
  if (gemm_tiles(a0)) return launch_linear_gemm(a0, a, st);
  const Plan p = plan(a0);
  const bool g = lin_gated(a.activation);
  if (a.x_dtype == MI355MOE_FP8E4M3 && a0.out_dtype == MI355MOE_F32)
    return g ? launch_tiles<K_FP8_EXACT, true>(a, p, st) : launch_tiles<K_FP8_EXACT, false>(a, p, st);
  if (a.x_dtype == MI355MOE_FP8E4M3)
    return g ? launch_tiles<K_FP8, true>(a, p, st) : launch_tiles<K_FP8, false>(a, p, st);
  if (a.x_dtype == MI355MOE_F16)
    return g ? launch_tiles<K_F16, true>(a, p, st) : launch_tiles<K_F16, false>(a, p, st);
  return g ? launch_tiles<K_BF16, true>(a, p, st) : launch_tiles<K_BF16, false>(a, p, st);
}

}  // namespace mi355
