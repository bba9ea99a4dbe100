// Attention over packed sequences of different lengths, forward: softmax(q k^T scale) v of every sequence of a batch in one launch, causal or
// not, with grouped heads.
//
// A workgroup takes 32 rows per wave of one sequence and one query head.  S^T = K Q^T and O^T += V^T P^T in 32x32x16 bf16 MFMAs over
// tiles of 64 keys that its waves share in LDS: a lane owns one query column, so the row maximum and sum of the softmax are in-lane
// reductions and one exchange with lane^32, and P^T is in the B operand's layout as it leaves the accumulators.  Iteration t issues the
// fills of K(t+2) and V(t+1), runs S(t+1) and then O += P(t) V(t) on the matrix cores while the vector ALU forms P(t) and then the row
// maximum of S(t+1); one barrier per tile.  The maximum that P refers to is only raised where a row grows by more than 2^8 (exact: numerator and
// denominator share it).  P is rounded to bf16 (2^-9 of each on average, and the errors of a row's keys are independent); its sum is not.
//
// Bound by the matrix cores at the clock that the power limit leaves, which differs from card to card: 32768 tokens of 32 heads over 8 of 128, causal, 7.1 to
// 7.6 ms, 1160 to 1240 TFLOP/s with the matrix cores busy 78 % of the cycles at 1.5 GHz; 16 ragged prompts of up to 4096 tokens 601 to 643 us, 960 to
// 1020 TFLOP/s (59 %), 12 sequences of up to 2047 150 us, 795 TFLOP/s (48 %): a tile of a few keys pays for its start and end.
// Every operand of a product is read from LDS, 1 KiB per product, which is what LDS gives
// at full rate; with half of the reads left out (and wrong results) the same launches take 5 % less, so wider waves would not pay.
#include "packed.h"

namespace lvar {

#if defined(__HIP_DEVICE_COMPILE__)

// A row of the output whose sums are not finite, key by key: 0 * infinity from a masked key's value must not stay in it.  M and L are
// those of the row (values do not enter them).  Rare, and so plain: lanes are keys for the scores, columns for the sums.
template <int D>
__device__ __forceinline__ void careful_row(const bf16_t* q, const bf16_t* k, int64_t k_sr, const bf16_t* v, int64_t v_sr, int seen, float c, float m,
                                         float inv, bf16_t* o) {
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  float acc[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; e++) acc[e] = 0.f;
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const int n = min(64, seen - j0);
    const bf16_t* kr = k + (int64_t)(j0 + min(lane, n - 1)) * k_sr;
    float s = 0.f;
    for (int e = 0; e < D; e++) s = fmaf((float)q[e], (float)kr[e], s);
    const float w = fast_exp2(fmaf(s, c, -m)) * inv;
    for (int j = 0; j < n; j++) {
      const float x = __shfl(w, j, 64);
#pragma unroll
      for (int e = 0; e < D / 64; e++) acc[e] = fmaf(x, (float)v[(int64_t)(j0 + j) * v_sr + e * 64 + lane], acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < D / 64; e++) o[e * 64 + lane] = (bf16_t)acc[e];
}

template <int D, int NW, bool SPLIT>
__device__ __forceinline__ void packed_fwd_item(const PackedParams& p, char* smem, const PackedTile& w, const int h, const int share) {
  using S = PackedLds<D>;
  constexpr int KS = D / 16, MTD = D / 32, ROWS = NW * 32, TILE = S::TILE, SLOTS = S::NI / NW;
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  const int wave = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_workitem_id_x() >> 6);
  const int hh = lane >> 5, r = lane & 31;
  const S at(lane);
  const int m_all = w.other_n;
  const int hk = h / p.G, q0 = w.row0 + wave * 32;   // first row of the wave
  const int shift = p.causal ? m_all - w.n : m_all;  // row i sees keys below i + shift + 1 (causal), below m_all
  auto all_seen_by = [&](int row) { return max(0, p.causal ? min(m_all, row + shift + 1) : m_all); };
  const int T_all = (all_seen_by(min(w.row0 + ROWS, w.n) - 1) + 63) >> 6;
  const Share part = SPLIT ? share_of(T_all, share, p.shares) : Share{0, T_all};
  // from here on keys are those of the share
  const int T = part.T, k_first = w.other_first + 64 * part.t0, m = SPLIT ? max(0, min(m_all - 64 * part.t0, 64 * T)) : m_all;
  auto seen_by = [&](int row) { return SPLIT ? max(0, min(m, all_seen_by(row) - 64 * part.t0)) : all_seen_by(row); };
  const int row = min(q0 + r, w.n - 1);
  const int seen = seen_by(row), seen_first = __builtin_amdgcn_readfirstlane(seen);   // lane 0 has the wave's first row: the fewest

  f32x16 oacc[MTD];
#pragma unroll
  for (int i = 0; i < MTD; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) oacc[i][e] = 0.f;
  float m_ref = NEG_BIG, m_true = -INFINITY, lsum[2] = {0.f, 0.f};
  const float c = p.c;
  const bf16_t* qp = p.q + h * p.q_sh + (int64_t)(w.first + row) * p.q_sr;
  const bf16_t *kp = p.k + hk * p.k_sh + (int64_t)k_first * p.k_sr, *vp = p.v + hk * p.v_sh + (int64_t)k_first * p.v_sr;

  if (T > 0) {
    const int k_srb = (int)p.k_sr * 2, v_srb = (int)p.v_sr * 2;
    const i32x4 krsrc = packed_rsrc(kp, m, S::ROWB, k_srb), vrsrc = packed_rsrc(vp, m, S::ROWB, v_srb);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(LVAR_LDS char*)smem;
    // K buffers at 0 and TILE, V buffers at 2 TILE and 3 TILE
    fill_tile<D, NW>(krsrc, k_srb, 0, lds0, wave, lane);
    fill_tile<D, NW>(vrsrc, v_srb, 0, lds0 + 2 * TILE, wave, lane);
    if (T > 1) fill_tile<D, NW>(krsrc, k_srb, 64, lds0 + TILE, wave, lane);
    bf16x8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) qf[ks] = *(const bf16x8*)(qp + hh * 8 + ks * 16);
    wait_fills<0>();
    __syncthreads();

    // keys that a row does not see (accumulator i is key 8 (i / 4) + 4 hh + i % 4 of the tile, or 32 more)
    auto mask = [&](int t, f32x16& s0, f32x16& s1) {
      const int lim = seen - 64 * t - 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int kc = 8 * (i >> 2) + (i & 3);
        s0[i] = kc < lim ? s0[i] : -INFINITY;
        s1[i] = kc + 32 < lim ? s1[i] : -INFINITY;
      }
    };
    auto raise = [&](float mx) {
      const float mt = mx * c;
      m_true = fmaxf(m_true, mt);
      if (__builtin_amdgcn_ballot_w64(mt > m_ref + RESCALE_TAU) != 0) {
        const float m_new = fmaxf(m_ref, mt), alpha = fast_exp2(m_ref - m_new);
        lsum[0] *= alpha;
        lsum[1] *= alpha;
#pragma unroll
        for (int i = 0; i < MTD; i++)
#pragma unroll
          for (int e = 0; e < 16; e++) oacc[i][e] *= alpha;
        m_ref = m_new;
      }
    };

    f32x16 sa0, sa1, sb0, sb1;
#pragma unroll
    for (int i = 0; i < 16; i++) { sa0[i] = 0.f; sa1[i] = 0.f; }
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      sa0 = mfma32(at.rows(smem, 0, ks), qf[ks], sa0);
      sa1 = mfma32(at.rows(smem, 1, ks), qf[ks], sa1);
    }
    __syncthreads();   // all have read K(0): K(2) takes its place
    if (seen_first < 64) mask(0, sa0, sa1);
    {
      float ma = fmaxf(sa0[0], sa1[0]);
#pragma unroll
      for (int i = 1; i < 16; i++) ma = fmaxf(fmaxf(ma, sa0[i]), sa1[i]);
      raise(xhalf_max(ma));
    }

    // Tile t, which has a successor, PAR = t & 1: K(t+1) is in K buffer 1 - PAR, V(t) in V buffer PAR.  Straight-line code, held in its order by
    // scheduling barriers: QK MFMA j beside the read of operand j + 4 and softmax slot j of S(t), then PV MFMA j beside the last slots
    // and the row maximum of S(t+1).  A slot scales its elements, takes exp2 of those of the slot before, and adds and packs those
    // before that, so that no vector instruction waits for the one before it.
    auto body = [&](int t, auto par, auto has_mask, f32x16& c0, f32x16& c1, f32x16& n0, f32x16& n1) {
      constexpr int PAR = decltype(par)::value, NQK = 2 * KS, NPV = 4 * MTD, AHEAD = READ_AHEAD, HB = NPV / 2;
      constexpr bool MASKED = decltype(has_mask)::value;
      constexpr int NFILL = 2 * SLOTS, FSTRIDE = NFILL <= NQK ? NQK / NFILL : 1, PER = (NFILL + NQK - 1) / NQK;
      const char *kbuf = smem + (1 - PAR) * TILE, *vbuf = smem + (2 + PAR) * TILE;
      auto fill_step = [&](auto jc) {
        constexpr int j = decltype(jc)::value;
        if constexpr (j % FSTRIDE == 0) {
#pragma unroll
          for (int f = j / FSTRIDE * PER; f < (j / FSTRIDE + 1) * PER; f++) {
            if (f < SLOTS) fill_slot<D, NW>(vrsrc, v_srb, 64 * (t + 1), lds0 + (3 - PAR) * TILE, wave, lane, f);
            else if (f < NFILL) fill_slot<D, NW>(krsrc, k_srb, 64 * (t + 2), lds0 + PAR * TILE, wave, lane, f - SLOTS);
          }
        }
      };
      bf16x8 frag[NQK > NPV ? NQK : NPV];
      uint32_t pw[16];
      const float negm = -m_ref;
      float la = 0.f, lb = 0.f;
      auto st_scale = [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (e < 16) c0[e] = fmaf(c0[e], c, negm); else c1[e - 16] = fmaf(c1[e - 16], c, negm);
      };
      auto st_exp = [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (e < 16) c0[e] = fast_exp2(c0[e]); else c1[e - 16] = fast_exp2(c1[e - 16]);
      };
      auto st_sum = [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        float x;
        if constexpr (e < 16) x = c0[e]; else x = c1[e - 16];
        if constexpr (e < 16) la += x; else lb += x;
        if constexpr (e == 15) lsum[0] += la;
        if constexpr (e == 31) lsum[1] += lb;
        if constexpr (e & 1) {
          float prev;
          if constexpr (e < 16) prev = c0[e - 1]; else prev = c1[e - 17];
          pw[e >> 1] = pack_bf16(prev, x);
        }
      };
      using Sch = ExpSlots<NQK, HB, EXP_IN_QK>;
      auto softmax_step = [&](auto gc) {
        constexpr int g = decltype(gc)::value;
        static_for<Sch::lo(g - 2), Sch::lo(g - 1)>(st_sum);
        static_for<Sch::lo(g - 1), Sch::lo(g)>(st_exp);
        static_for<Sch::lo(g), Sch::lo(g + 1)>(st_scale);
      };
#pragma unroll
      for (int j = 0; j < AHEAD; j++) frag[j] = at.rows(kbuf, j & 1, j >> 1);
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, NQK>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        if constexpr (j + AHEAD < NQK) frag[j + AHEAD] = at.rows(kbuf, (j + AHEAD) & 1, (j + AHEAD) >> 1);
        if constexpr (j == 0) n0 = mfma32(frag[j], qf[0], f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0});
        else if constexpr (j == 1) n1 = mfma32(frag[j], qf[0], f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0});
        else if constexpr (j & 1) n1 = mfma32(frag[j], qf[j >> 1], n1);
        else n0 = mfma32(frag[j], qf[j >> 1], n0);
        fill_step(jc);
        softmax_step(jc);
        __builtin_amdgcn_sched_barrier(0);
      });
      float ma = -INFINITY;
      bf16x8 pb[4];
#pragma unroll
      for (int j = 0; j < AHEAD; j++) frag[j] = at.columns(vbuf, j / MTD, j % MTD);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MASKED) mask(t + 1, n0, n1);
      static_for<0, NPV>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        if constexpr (j + AHEAD < NPV) frag[j + AHEAD] = at.columns(vbuf, (j + AHEAD) / MTD, (j + AHEAD) % MTD);
        if constexpr (j % MTD == 0) {
          constexpr int kb = j / MTD;
          const u32x4 u = {pw[4 * kb], pw[4 * kb + 1], pw[4 * kb + 2], pw[4 * kb + 3]};
          pb[kb] = __builtin_bit_cast(bf16x8, u);
        }
        oacc[j % MTD] = mfma32(frag[j], pb[j / MTD], oacc[j % MTD]);
        softmax_step(std::integral_constant<int, NQK + j>{});
        if constexpr (j >= HB) {
          constexpr int e0 = (j - HB) * 16 / (NPV - HB), e1 = (j - HB + 1) * 16 / (NPV - HB);
#pragma unroll
          for (int e = e0; e < e1; e++) ma = fmaxf(fmaxf(ma, n0[e]), n1[e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      const float mx = xhalf_max(ma);
      wait_fills<0>();
      __syncthreads();
      raise(mx);
    };
    auto last = [&](auto par, f32x16& c0, f32x16& c1) {
      constexpr int PAR = decltype(par)::value;
      const char* vbuf = smem + (2 + PAR) * TILE;
      bf16x8 pb[4];
#pragma unroll
      for (int i = 0; i < 16; i++) {
        c0[i] = fast_exp2(fmaf(c0[i], c, -m_ref));
        c1[i] = fast_exp2(fmaf(c1[i], c, -m_ref));
        lsum[0] += c0[i];
        lsum[1] += c1[i];
      }
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        pb[kb] = pack8(c0[8 * kb], c0[8 * kb + 1], c0[8 * kb + 2], c0[8 * kb + 3], c0[8 * kb + 4], c0[8 * kb + 5], c0[8 * kb + 6], c0[8 * kb + 7]);
        pb[kb + 2] = pack8(c1[8 * kb], c1[8 * kb + 1], c1[8 * kb + 2], c1[8 * kb + 3], c1[8 * kb + 4], c1[8 * kb + 5], c1[8 * kb + 6], c1[8 * kb + 7]);
      }
#pragma unroll
      for (int kb = 0; kb < 4; kb++)
#pragma unroll
        for (int i = 0; i < MTD; i++) oacc[i] = mfma32(at.columns(vbuf, kb, i), pb[kb], oacc[i]);
    };
    using P0 = std::integral_constant<int, 0>;
    using P1 = std::integral_constant<int, 1>;
    using No = std::false_type;
    using Yes = std::true_type;
    // tiles that all rows of the wave see whole, then the others that one of them sees (loops of their own: behind a branch in one loop the two
    // bodies spill), then those that only other waves do
    const int mine = q0 < w.n ? (seen_by(min(q0 + 32, w.n) - 1) + 63) >> 6 : 0, whole = min(mine, seen_first >> 6);
    int t = 0;
    for (; t + 2 < whole; t += 2) {
      body(t, P0{}, No{}, sa0, sa1, sb0, sb1);
      body(t + 1, P1{}, No{}, sb0, sb1, sa0, sa1);
    }
    for (; t + 2 < mine; t += 2) {
      body(t, P0{}, Yes{}, sa0, sa1, sb0, sb1);
      body(t + 1, P1{}, Yes{}, sb0, sb1, sa0, sa1);
    }
    if (t + 1 < mine) {
      body(t, P0{}, Yes{}, sa0, sa1, sb0, sb1);
      last(P1{}, sb0, sb1);
    } else if (mine > 0) {
      last(P0{}, sa0, sa1);
    }
    for (t = max(0, mine - 1); t + 1 < T; t++) {
      fill_tile<D, NW>(vrsrc, v_srb, 64 * (t + 1), lds0 + (2 + ((t + 1) & 1)) * TILE, wave, lane);
      fill_tile<D, NW>(krsrc, k_srb, 64 * (t + 2), lds0 + (t & 1) * TILE, wave, lane);
      wait_fills<0>();
      __syncthreads();
    }
    __syncthreads();
  }

  const float ltot = xhalf_sum(lsum[0] + lsum[1]);
  const bool empty = bits_of(ltot) == 0u;   // no key seen
  if constexpr (SPLIT) {   // packed_fwd_join_kernel does the rest
    const int64_t at_row = ((int64_t)share * p.H + h) * p.T + w.first + q0;
    if (hh == 0 && q0 + r < w.n) {
      float* st = p.part_stats + (at_row + r) * 3;
      st[0] = m_ref;
      st[1] = ltot;
      st[2] = m_true;
    }
    if (T > 0) store_part<D>(smem + wave * (32 * (D * 2 + 16)), oacc, p.parts + at_row * D, w.n - q0, lane);
    return;
  }
  const float inv = empty ? 0.f : 1.0f / ltot;
  if (hh == 0 && q0 + r < w.n) {
    const int64_t to = (int64_t)h * p.T + w.first + q0 + r;
    p.M[to] = empty ? -INFINITY : m_true;
    p.L[to] = empty ? 1.0f : ltot * fast_exp2(m_ref - m_true);
  }
  bf16_t* op = p.o + h * p.o_sh + (int64_t)(w.first + q0) * p.o_sr;
  store_rows<D>(smem + wave * (32 * (D * 2 + 16)), oacc, inv, op, p.o_sr, w.n - q0, lane);
  if (p.causal) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < MTD; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) bad |= not_finite(oacc[i][e]);
    uint64_t rows = __builtin_amdgcn_ballot_w64(bad && q0 + r < w.n);
    rows = (rows | rows >> 32) & 0xffffffffu;
    if (rows) wait_fills<0>();   // the rows as stored above are written again
    while (rows) {
      const int i = __builtin_ctzll(rows);
      rows &= rows - 1;
      const float mi = __shfl(m_ref, i, 64), ii = __shfl(inv, i, 64);
      careful_row<D>(p.q + h * p.q_sh + (int64_t)(w.first + q0 + i) * p.q_sr, kp, p.k_sr, vp, p.v_sr, __shfl(seen, i, 64), c, mi, ii, op + i * p.o_sr);
    }
  }
}

#endif  // __HIP_DEVICE_COMPILE__

template <int D, int NW>
constexpr int packed_fwd_lds() {
  const int bufs = 4 * 64 * D * 2, out = NW * 32 * (D * 2 + 16);
  return bufs > out ? bufs : out;
}

template <int D, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void packed_fwd_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int per = SPLIT ? p.H * p.shares : p.H;
  const int id = __builtin_amdgcn_workgroup_id_x(), place = id / per, j = id - place * per;
  PackedTile w;
  // the places from the last one on: of a causal sequence the tiles with the most keys come first
  if (!find_tile<NW * 32>(p.q_off, p.T, p.k_off, p.Tk, p.B, p.slots - 1 - place, false, w)) return;
  const int share = SPLIT ? j / p.H : 0;
  packed_fwd_item<D, NW, SPLIT>(p, smem, w, packed_head(j - share * p.H, p.H), share);
#endif
}

// The rows of a launch whose workgroups shared keys, from the parts in their order: a lane per four columns.
template <int D>
__global__ __launch_bounds__(256) void packed_fwd_join_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int LPR = D / 4, RPG = 256 / LPR;
  const int tid = __builtin_amdgcn_workitem_id_x(), lane = tid & 63, column = tid % LPR * 4;
  const int64_t rows = (int64_t)p.H * p.T, x = (int64_t)__builtin_amdgcn_workgroup_id_x() * RPG + tid / LPR, at = min(x, rows - 1);
  const int h = (int)(at / p.T), row = (int)(at - (int64_t)h * p.T);
  const float *st = p.part_stats + at * 3, *part = p.parts + at * D + column;
  float M = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < p.shares; s++) M = fmaxf(M, st[s * rows * 3 + 2]);
  float L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  bool any = false;
  for (int s = 0; s < p.shares; s++) {
    const float sum = st[s * rows * 3 + 1];
    const f32x4 y = *(const f32x4*)(part + s * rows * D);
    const bool some = bits_of(sum) != 0u;   // a key of the share is seen (else its part may not be written)
    any |= some;
    const float f = some ? fast_exp2(st[s * rows * 3] - M) : 0.f;
    L = fmaf(f, sum, L);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = fmaf(f, some ? y[e] : 0.f, o[e]);
  }
  const float inv = any ? 1.0f / L : 0.f;
  bf16_t* to = p.o + h * p.o_sh + (int64_t)row * p.o_sr;
  if (x < rows) {
    if (column == 0) {
      p.M[at] = any ? M : -INFINITY;
      p.L[at] = any ? L : 1.0f;
    }
    *(u32x2*)(to + column) = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
  }
  if (!p.causal) return;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad |= not_finite(o[e]);
  uint64_t left = __builtin_amdgcn_ballot_w64(bad && x < rows);
  if (left) wait_fills<0>();   // the rows as stored above are written again
  while (left) {
    const int i = __builtin_ctzll(left) / LPR * LPR;   // the first lane of a row
    left &= i + LPR < 64 ? ~0ull << (i + LPR) : 0ull;
    const int hi = __builtin_amdgcn_readlane(h, i), ri = __builtin_amdgcn_readlane(row, i), hk = hi / p.G;
    PackedTile w;
    find_row(p.q_off, p.T, p.k_off, p.Tk, p.B, ri, w);
    const int seen = max(0, min(w.other_n, w.row0 + w.other_n - w.n + 1));
    careful_row<D>(p.q + hi * p.q_sh + (int64_t)ri * p.q_sr, p.k + hk * p.k_sh + (int64_t)w.other_first * p.k_sr, p.k_sr,
                   p.v + hk * p.v_sh + (int64_t)w.other_first * p.v_sr, p.v_sr, seen, p.c, __shfl(M, i, 64), __shfl(inv, i, 64), p.o + hi * p.o_sh + (int64_t)ri * p.o_sr);
  }
#endif
}

template <int D, int NW, bool SPLIT>
static int launch_fwd(PackedParams p, hipStream_t s) {
  constexpr int SMEM = packed_fwd_lds<D, NW>();
  const int64_t slots = packed_slots(p.T, p.B, NW * 32), groups = slots * p.H * p.shares, joins = ((int64_t)p.H * p.T * (D / 4) + 255) / 256;
  if (groups * (NW * 64) > 0xffffffffll || (SPLIT && joins * 256 > 0xffffffffll)) return LVAR_EINVAL;
  p.slots = (int)slots;
  auto kern = packed_fwd_kernel<D, NW, SPLIT>;
  static std::atomic<uint64_t> ready{0};
  if (!ensure_lds_limit((const void*)kern, SMEM, ready)) return LVAR_ELAUNCH;
  hipLaunchKernelGGL(kern, dim3((uint32_t)groups), dim3(NW * 64), SMEM, s, p);
  if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (SPLIT) hipLaunchKernelGGL(packed_fwd_join_kernel<D>, dim3((uint32_t)joins), dim3(256), 0, s, p);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

static int fwd_shares(const PackedParams& p, int head_dim) { return query_shares(p, head_dim <= 128 ? 2 : 1); }

// sums and statistics of shares
int64_t packed_fwd_bytes(const PackedParams& p, int head_dim) {
  const int shares = fwd_shares(p, head_dim);
  return shares > 1 ? 4 * (int64_t)shares * p.H * p.T * (head_dim + 3) : 0;
}

int launch_packed_fwd(PackedParams p, void* workspace, int head_dim, hipStream_t s) {
  p.shares = fwd_shares(p, head_dim);
  p.parts = (float*)workspace;
  p.part_stats = p.parts + (int64_t)p.shares * p.H * p.T * head_dim;
  const bool split = p.shares > 1;
  if (head_dim == 128) return split ? launch_fwd<128, 4, true>(p, s) : launch_fwd<128, 4, false>(p, s);
  if (head_dim == 64) return split ? launch_fwd<64, 4, true>(p, s) : launch_fwd<64, 4, false>(p, s);
  if (head_dim == 256) return split ? launch_fwd<256, 4, true>(p, s) : launch_fwd<256, 4, false>(p, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
