// The body of gemm_tile_kernel, and of what runs two products in one launch: the tiles of `walk`, of
// `a`'s product, through the ring `lds`.  Its template arguments are gemm_tile_kernel's.  It is included
// as text: inlined from a function, the compiler keeps 41 more registers through the int8 epilogue
// (128 x 256: 215 -> 256 and 13 in scratch; 8192 x 2048 x 7168 174 -> 182 us, 4096^3 79 -> 83).
  constexpr bool I8 = KIND == K_I8;
  constexpr int EB = kind_bytes(KIND);
  static_assert(!(I8 && (TQ || TP)) && !(GATED && TP) && !(TQ && !TP), "operands");
  constexpr int WAVES = WI * WJ, THREADS = 64 * WAVES;
  constexpr int MT = BI / WI / 32, NT = BJ / WJ / 32;
  constexpr int NO = GATED ? NT / 2 : NT;                     // tiles of outputs
  static_assert(MT >= 1 && NO >= 1 && (!GATED || NT % 2 == 0), "wave tile");
  constexpr int BJO = GATED ? BJ / 2 : BJ;                    // output columns
  constexpr int BR = GSB / EB;                                // r of a stage
  constexpr int STAGE = (BI + BJ) * GSB;
  constexpr int QCH = TQ ? BI / 8 : 8, PCH = TP ? BJ / 8 : 8;  // 16-byte chunks of a staged row
  constexpr int QQ = BI / 8 / WAVES, PQ = BJ / 8 / WAVES, ND = QQ + PQ;  // copies per wave and stage
  static_assert(QQ * 8 * WAVES == BI && PQ * 8 * WAVES == BJ, "copies");
  static_assert(!GATED || PQ % 2 == 0, "a copy has rows of one half");
  constexpr bool LIN = EPI == E_LINEAR || EPI == E_KEEP;
  float* s_bias = reinterpret_cast<float*>(lds + NSTAGE * STAGE);  // [BJ]
  float* s_ws = s_bias + BJ;                                       // [BJ]
  float* s_xs = s_ws + BJ;                                         // [BI]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave / WJ, wj = wave % WJ;
  const int g4 = lane >> 4, t16 = lane & 15, h = lane >> 5, l32 = lane & 31;

  if (walk.t >= walk.end) return;  // uniform

  // p's rows (along r) of weight tile i, and its columns in the output
  auto prow = [&](int i) __attribute__((always_inline)) {
    if constexpr (GATED)
      return i < NO ? wj * (BJO / WJ) + 32 * i : BJO + wj * (BJO / WJ) + 32 * (i - NO);
    else
      return wj * (BJ / WJ) + 32 * i;
  };

  // ---- a tile: its place, its stages, its copies' offsets
  int64_t i0, j0;
  int split, k0, nk, tail;  // tail: r of the last stage, 0: all
  uint64_t qbase, pbase;
  uint32_t voff[ND];
  const uint64_t qstep = TQ ? static_cast<uint64_t>(a.ldx) * (2 * BR) : GSB;
  const uint64_t pstep = TP ? static_cast<uint64_t>(a.ldw) * (2 * BR) : GSB;
  const uint64_t uhalf = GATED ? static_cast<uint64_t>(a.N) * a.ldw * EB : 0;
  // the 16 bytes that this lane copies: their number in the staged operand
  auto piece_of = [=](int q) __attribute__((always_inline)) {
    if (q < QQ) return (wave * QQ + q) * 64 + lane;
    // (gated: a wave's first copies are the gate's rows, its others the factor's)
    if (GATED) return (wave * (PQ / 2) + (q - QQ) % (PQ / 2)) * 64 + lane;
    return (wave * PQ + q - QQ) * 64 + lane;
  };
  auto row_of = [=](int q) __attribute__((always_inline)) { return piece_of(q) / (q < QQ ? QCH : PCH); };
  auto place = [&](int tile) __attribute__((always_inline)) {
    split = tile / (tiles_i * tiles_j);
    tile %= tiles_i * tiles_j;
    constexpr int band_rows = 4;
    const int band = tile / (band_rows * tiles_j);
    const int bi = tiles_i - band * band_rows < band_rows ? tiles_i - band * band_rows : band_rows;
    tile -= band * band_rows * tiles_j;
    i0 = static_cast<int64_t>(band * band_rows + tile % bi) * BI;
    j0 = static_cast<int64_t>(tile / bi) * BJO;
    const int nk_all = static_cast<int>((a.K + BR - 1) / BR);
    k0 = split * stages_per_split;
    nk = nk_all - k0 < stages_per_split ? nk_all - k0 : stages_per_split;
    tail = k0 + nk == nk_all ? static_cast<int>(a.K % BR) : 0;
    qbase = uniform64(reinterpret_cast<uint64_t>(a.x) + static_cast<uint64_t>((TQ ? i0 : i0 * a.ldx) * EB) + k0 * qstep);
    pbase = uniform64(reinterpret_cast<uint64_t>(a.weight) + static_cast<uint64_t>((TP ? j0 : j0 * a.ldw) * EB) + k0 * pstep);
    // (rows across r are readable to a multiple of 8 columns)
    const int qlast = static_cast<int>(((a.M + 7) / 8 - i0 / 8 < QCH ? (a.M + 7) / 8 - i0 / 8 : QCH) - 1);
    const int plast = static_cast<int>(((a.N + 7) / 8 - j0 / 8 < PCH ? (a.N + 7) / 8 - j0 / 8 : PCH) - 1);
#pragma unroll
    for (int q = 0; q < ND; ++q) {
      const int r = row_of(q);
      const bool x = q < QQ;
      const int64_t ld = x ? a.ldx : a.ldw;
      if (x ? TQ : TP) {
        const int c = x ? (piece_of(q) % QCH) ^ cross_swz<QCH>(r) : (piece_of(q) % PCH) ^ cross_swz<PCH>(r);
        const int last = x ? qlast : plast;
        voff[q] = static_cast<uint32_t>(r * ld * EB + ((c < last ? c : last) << 4));
      } else {
        const int64_t last = x ? a.M - 1 - i0 : a.N - 1 - j0;
        voff[q] = static_cast<uint32_t>((r < last ? r : last) * ld * EB + (((lane % 8) ^ gswz(r)) << 4));
      }
    }
  };

  const uint32_t ring = lds_off(lds);
  // copy Q into the slot at LDS offset `slot`; past: the stage holds `tail` r, rows behind
  // them repeat the last, chunks behind them the stage's first
  auto copy = [&](auto qc, uint64_t qoff, uint64_t poff, uint32_t slot, bool past)
      __attribute__((always_inline)) {
    constexpr int Q = decltype(qc)::value;
    constexpr bool X = Q < QQ;
    constexpr bool UP = GATED && !X && Q - QQ >= PQ / 2;
    uint32_t v = voff[Q];
    if (past) {  // uniform
      const int r = row_of(Q);
      if constexpr (X ? TQ : TP) {
        if (r >= tail) v -= static_cast<uint32_t>((r - (tail - 1)) * (X ? a.ldx : a.ldw) * EB);
      } else {
        const int cb = ((lane % 8) ^ gswz(r)) << 4;
        if (cb >= EB * tail) v -= cb;
      }
    }
    if constexpr (X) dma16<Q * 1024>(v, qbase + qoff, slot + wave * (QQ * 1024));
    else if constexpr (GATED)
      dma16<BI * GSB + (UP ? BJO * GSB : 0) + ((Q - QQ) % (PQ / 2)) * 1024>(
          v, pbase + poff + (UP ? uhalf : 0), slot + wave * (PQ / 2 * 1024));
    else dma16<BI * GSB + (Q - QQ) * 1024>(v, pbase + poff, slot + wave * (PQ * 1024));
  };
  auto issue = [&](int kt) __attribute__((always_inline)) {
    const uint32_t slot = ring + (kt % NSTAGE) * STAGE;
    const bool past = tail != 0 && kt == nk - 1;
    for_each<ND>([&](auto q) __attribute__((always_inline)) {
      copy(q, static_cast<uint64_t>(kt) * qstep, static_cast<uint64_t>(kt) * pstep, slot, past);
    });
  };
  auto first_stages = [&]() __attribute__((always_inline)) {
    for (int s = 0; s < NSTAGE && s < nk; ++s) issue(s);
  };
  // the last stage's r behind `tail` (along r: whole chunks; a dz row holds zeros up to one)
  auto clear_tail = [&](int kt) __attribute__((always_inline)) {
    uint8_t* S = lds + (kt % NSTAGE) * STAGE;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto along = [&](uint8_t* s, int rows) __attribute__((always_inline)) {
      for (int i = tid; i < rows * 8; i += THREADS) {
        const int r = i >> 3, c = i & 7;
        if ((c << 4) >= EB * tail) *reinterpret_cast<uint4*>(s + r * GSB + ((c ^ gswz(r)) << 4)) = zero;
      }
    };
    auto across = [&](uint8_t* s, int ch) __attribute__((always_inline)) {
      for (int i = tail * ch + tid; i < BR * ch; i += THREADS) reinterpret_cast<uint4*>(s)[i] = zero;
    };
    if constexpr (TQ) across(S, QCH);
    else along(S, BI);
    if constexpr (TP) across(S + BI * GSB, PCH);
    else along(S + BI * GSB, BJ);
    lds_barrier();
  };
  // publishes stage kt + 1; every wave has read stage kt then
  auto advance = [&](int kt) __attribute__((always_inline)) {
    if (kt + 1 >= nk) return;
    if (kt + NSTAGE <= nk) wait_vm<ND * (NSTAGE - 2)>();
    else wait_vm<0>();
    lds_barrier();
    if (tail && kt + 2 == nk) clear_tail(kt + 1);
  };

  // Where this lane reads fragment n of an operand: across r, row 8 h + t / 4 (then + 4) of
  // a step, 4 columns from 16 (g & 1) + 4 (t & 3) of the fragment's 32; along r, chunk h of
  // row l32.
  auto cross_at = [&](auto ch, int col) __attribute__((always_inline)) {
    constexpr int CH = decltype(ch)::value;
    const int r = 8 * h + (t16 >> 2);
    return r * (CH * 16) + (((col / 8) ^ cross_swz<CH>(r)) << 4) +
           ((2 * (g4 & 1) + ((t16 & 3) >> 1)) << 4) + 8 * (t16 & 1);
  };
  int pat[NT], qat[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    pat[i] = BI * GSB + (TP ? cross_at(std::integral_constant<int, PCH>{}, wj * (BJ / WJ) + 32 * i)
                            : (prow(i) + l32) * GSB);
#pragma unroll
  for (int j = 0; j < MT; ++j)
    qat[j] = TQ ? cross_at(std::integral_constant<int, QCH>{}, wi * (BI / WI) + 32 * j)
                : (wi * (BI / WI) + 32 * j + l32) * GSB;
  const int sw = gswz(l32);

  constexpr int KS = 4;  // steps of 32 bytes along r
  struct Frag {
    uint4 q[MT], p[NT];
  };
  constexpr int NF = MT + NT;
  auto cross8 = [&](const uint8_t* s, int row) __attribute__((always_inline)) {
    const uint2 lo = lds_column4(s), hi = lds_column4(s + 4 * row);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  auto read = [&](Frag& o, const uint8_t* S, int ks, int e) __attribute__((always_inline)) {
    const int c = ((2 * ks + h) ^ sw) << 4;
    if (e == 0 || e > MT) {
      const int i = e == 0 ? 0 : e - MT;
      if constexpr (TP) o.p[i] = cross8(S + pat[i] + ks * (16 * PCH * 16), PCH * 16);
      else o.p[i] = lds16(S + pat[i] + c);
    } else {
      if constexpr (TQ) o.q[e - 1] = cross8(S + qat[e - 1] + ks * (16 * QCH * 16), QCH * 16);
      else o.q[e - 1] = lds16(S + qat[e - 1] + c);
    }
  };
  using Acc = typename SumVec<KIND, 16>::T;
  Acc acc[NT][MT];
  constexpr int NM = NT * MT, RPM = (NF + NM - 1) / NM, CPM = (ND + NM - 1) / NM;
  // One step: its MFMAs, between them the reads of the next step's fragments and, with
  // `dma`, the copies of a stage; the order is kept.
  auto step = [&](auto last_c, bool dma, const Frag& c, Frag& next, const uint8_t* Sn, int kn,
                  uint64_t qoff, uint64_t poff, uint32_t slot) __attribute__((always_inline)) {
    for_each<NM>([&](auto tc) __attribute__((always_inline)) {
      constexpr int m = decltype(tc)::value, i = m / MT, j = m % MT;
      acc[i][j] = mfma_32x32<KIND>(c.p[i], c.q[j], acc[i][j]);
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

  place(walk.t);
  first_stages();
  enum { NONE, SOME, WHOLE } behind = NONE;  // stores of the tile before
  for (;;) {
    // Stage 0 is there.  A whole tile's stores, issued behind these copies, may still be on
    // their way: one at least for each of the wave's runs.
    constexpr int LATER = ND * (NSTAGE - 1);
    if (nk < NSTAGE || behind == SOME) wait_vm<0>();
    else if (behind == NONE) wait_vm<LATER>();
    else wait_vm<(LATER + 2 * NO * MT < 63 ? LATER + 2 * NO * MT : 63)>();
    lds_barrier();
    if (tail && nk == 1) clear_tail(0);
    // biases and scales of this tile: every wave is done with the last one's
    if constexpr (LIN) {
      for (int i = tid; i < BJ; i += THREADS) {
        const bool up = GATED && i >= BJO;
        int64_t n = j0 + (up ? i - BJO : i);
        n = (n < a.N ? n : a.N - 1) + (up ? a.N : 0);
        s_bias[i] = a.bias ? ld_any(a.bias, a.bias_dtype, n) : 0.f;
        if constexpr (I8) s_ws[i] = w_scale_of(a, n);
      }
      if constexpr (I8)
        for (int i = tid; i < BI; i += THREADS) s_xs[i] = x_scale_of(a, i0 + i < a.M ? i0 + i : a.M - 1);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    {
      Frag f[2];
#pragma unroll
      for (int e = 0; e < NF; ++e) read(f[0], lds, 0, e);
      const int nfull = tail ? nk - 1 : nk;
      uint64_t qoff = NSTAGE * qstep, poff = NSTAGE * pstep;
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
    }
    const int64_t ti = i0, tj = j0;
    const int tsplit = split;
    const bool more = walk.more();  // uniform
    behind = ti + BI <= a.M && tj + BJO <= a.N ? WHOLE : SOME;
    lds_barrier();  // every wave has read the ring; biases and scales are there
    walk.next();

    // ---- epilogue
    const int xrow = wi * (BI / WI) + t16, xcol = 16 * (g4 & 1) + 8 * (g4 >> 1);  // see pair16
    if constexpr (!LIN) {
      if (more) {
        place(walk.t);
        first_stages();
      }
      const int64_t part = static_cast<int64_t>(tsplit) * a.M * a.N;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int64_t m = ti + xrow + 32 * j, n = tj + prow(i) + xcol;
          uint32_t v[2][8];
          gather8(acc[i][j], 0, v[0]);
          gather8(acc[i][j], 1, v[1]);
          if constexpr (EPI == E_PLAIN) {
            uint32_t w[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[e][k] = pack16x2<KIND == K_F16>(__uint_as_float(v[e][2 * k]), __uint_as_float(v[e][2 * k + 1]));
            pair16(w[0], w[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (m + 16 * e >= a.M) continue;
              uint16_t* o = static_cast<uint16_t*>(a.out) + (m + 16 * e) * a.ldo + n;
              if (n + 8 <= a.N) {
                put16(o, w[e][0], w[e][1], w[e][2], w[e][3]);
              } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  if (n + k < a.N) o[k] = static_cast<uint16_t>(w[e][k >> 1] >> (16 * (k & 1)));
              }
            }
          } else {
            pair16(v[0], v[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (m + 16 * e >= a.M) continue;
              uint32_t* o = static_cast<uint32_t*>(a.out) + part + (m + 16 * e) * a.N + n;
              if (n + 8 <= a.N) {
                put16(o, v[e][0], v[e][1], v[e][2], v[e][3]);
                put16(o + 4, v[e][4], v[e][5], v[e][6], v[e][7]);
              } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  if (n + k < a.N) o[k] = v[e][k];
              }
            }
          }
        }
    } else {
      const bool early = a.residual && a.residual_dtype != MI355MOE_F32 && tj + BJO <= a.N;
      // Residuals: all at once where 8 runs of 16 bytes hold them, else one row of tiles
      // ahead (memory operations end in order: a load behind stores waits for them).
      constexpr int RUNS = 2 * NO;
      constexpr bool ALL = RUNS * MT <= 8;
      uint32_t res[ALL ? MT : 2][RUNS][4];
      auto load_res = [&](uint32_t (&r)[RUNS][4], int j) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < RUNS; ++e) {
          int64_t m = ti + xrow + 32 * j + 16 * (e & 1);
          m = m < a.M ? m : a.M - 1;
          const any16_t v = *reinterpret_cast<const any16_t*>(static_cast<const uint16_t*>(a.residual) +
                                                              m * a.ldr + tj + prow(e >> 1) + xcol);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[e][k] = v[k];
        }
      };
      if (early) {
#pragma unroll
        for (int j = 0; j < (ALL ? MT : 1); ++j) load_res(res[j], j);
      }
      if (more) {
        place(walk.t);
        first_stages();
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (!ALL && early && j + 1 < MT) load_res(res[(j + 1) & 1], j + 1);
        const int row = wi * (BI / WI) + 32 * j + l32;
        const int64_t m = ti + row;
        const bool on = m < a.M;
        float xs = 0.f;
        if constexpr (I8) xs = s_xs[row];
#pragma unroll
        for (int i = 0; i < NO; ++i) {
          uint32_t (&r0)[4] = res[ALL ? j : j & 1][2 * i];
          uint32_t (&r1)[4] = res[ALL ? j : j & 1][2 * i + 1];
          if (early) pair16(r0, r1);
          float y[2][8];
          [[maybe_unused]] uint32_t kz[2][8], ku[2][8];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = prow(i) + 16 * e + 8 * h;
            const int64_t n = tj + c;
            float(&z)[8] = y[e];
            float u[8];
            auto sums = [&](const Acc& s, int col, float (&o)[8]) __attribute__((always_inline)) {
              uint32_t v[8];
              gather8(s, e, v);
              float b[8], w[8];
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float4 bb = *reinterpret_cast<const float4*>(s_bias + col + 4 * q);
                b[4 * q] = bb.x; b[4 * q + 1] = bb.y; b[4 * q + 2] = bb.z; b[4 * q + 3] = bb.w;
                if constexpr (I8) {
                  const float4 ww = *reinterpret_cast<const float4*>(s_ws + col + 4 * q);
                  w[4 * q] = ww.x; w[4 * q + 1] = ww.y; w[4 * q + 2] = ww.z; w[4 * q + 3] = ww.w;
                }
              }
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if constexpr (I8) o[k] = scaled_sum(static_cast<int>(v[k]), xs, w[k], b[k]);
                else o[k] = __uint_as_float(v[k]) + b[k];
              }
            };
            sums(acc[i][j], c, z);
            if constexpr (GATED) sums(acc[NO + i][j], BJO + c, u);
            if constexpr (EPI == E_KEEP) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                kz[e][k] = __float_as_uint(z[k]);
                ku[e][k] = __float_as_uint(u[k]);
              }
            }
            lin_act(a.activation, z);
            if constexpr (GATED) {
#pragma unroll
              for (int k = 0; k < 8; ++k) z[k] = times(z[k], u[k]);
            }
            if (early) {
              float r[8];
              const uint32_t(&rr)[4] = e ? r1 : r0;
              unpack8(make_uint4(rr[0], rr[1], rr[2], rr[3]), a.residual_dtype, r);
#pragma unroll
              for (int k = 0; k < 8; ++k) z[k] = plus(z[k], r[k]);
            } else if (a.residual) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (on && n + k < a.N) z[k] = plus(z[k], ld_any(a.residual, a.residual_dtype, m * a.ldr + n + k));
            }
          }
          const int64_t mx = ti + xrow + 32 * j, n = tj + prow(i) + xcol;
          // 8 floats of lane row mx + 16 e
          auto put = [&](float* o, const uint32_t (&v)[8]) __attribute__((always_inline)) {
            if (n + 8 <= a.N) {
              put16(o, v[0], v[1], v[2], v[3]);
              put16(o + 4, v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (n + k < a.N) o[k] = __uint_as_float(v[k]);
            }
          };
          if constexpr (EPI == E_KEEP) {
            pair16(kz[0], kz[1]);
            pair16(ku[0], ku[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (mx + 16 * e < a.M) {
                float* zo = a.z + (mx + 16 * e) * 2 * a.N + n;
                put(zo, kz[e]);
                put(zo + a.N, ku[e]);
              }
          }
          if (a.out_dtype == MI355MOE_F32) {
            uint32_t w[2][8];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int k = 0; k < 8; ++k) w[e][k] = __float_as_uint(y[e][k]);
            pair16(w[0], w[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (mx + 16 * e < a.M) put(static_cast<float*>(a.out) + (mx + 16 * e) * a.ldo + n, w[e]);
          } else {
            uint32_t w[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[e][k] = a.out_dtype == MI355MOE_BF16 ? pack16x2<false>(y[e][2 * k], y[e][2 * k + 1])
                                                       : pack16x2<true>(y[e][2 * k], y[e][2 * k + 1]);
            pair16(w[0], w[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (mx + 16 * e >= a.M) continue;
              uint16_t* o = static_cast<uint16_t*>(a.out) + (mx + 16 * e) * a.ldo + n;
              if (n + 8 <= a.N) {
                put16(o, w[e][0], w[e][1], w[e][2], w[e][3]);
              } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  if (n + k < a.N) o[k] = static_cast<uint16_t>(w[e][k >> 1] >> (16 * (k & 1)));
              }
            }
          }
        }
      }
    }
    if (!more) return;
  }
