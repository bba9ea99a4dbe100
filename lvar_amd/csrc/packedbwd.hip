// Attention over packed sequences, backward: with P = exp2(c s - M) / L, delta = sum(do * o) of a row and dS = P * (do v^T - delta),
//
//   dq = scale dS k        dk = scale dS^T q        dv = P^T do        (k and v: summed over the query heads that share them)
//
// in two launches, so that every sum is formed in one place and in a fixed order (no atomics): one over query tiles for dq, which also
// writes -(M + log2 L) / c and -delta of every row, and one over key tiles for dk and dv.  Both form s and do v^T again: seven products
// of (queries x keys x head_dim) instead of five, and no exchange of partial sums.  32x32x16 bf16 MFMAs with fp32 sums; P and dS are rounded to
// bf16 where they become operands (2^-9 of each on average; errors of a sum's terms are independent).
#include "packed.h"

namespace lvar {

#if defined(__HIP_DEVICE_COMPILE__)

// One row of a gradient whose sums are not finite, pair by pair: 0 * infinity from a row that does not see a key, or from the zeros behind the last row
// or key of a tile, must not stay in it.
// x0, x1: the fixed row (of q and do, or of k and v); y0, y1: the rows of the other side, lo .. hi-1.  ds weighs y0, P weighs y1 (KEY).
// Rare, and so plain: lanes are pairs for the products, columns for the sums.
template <int D, bool KEY>
struct CarefulRow {
  float a0[D / 64], a1[D / 64];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < D / 64; e++) a0[e] = a1[e] = 0.f;
  }
  // nl, nd: of the fixed row, or (KEY) of the rows on the other side
  __device__ __forceinline__ void add(const bf16_t* x0, const bf16_t* x1, const bf16_t* y0, int64_t y0_sr, const bf16_t* y1, int64_t y1_sr, int lo, int hi,
                                      const float* nl, const float* nd, float c) {
    const int lane = __builtin_amdgcn_workitem_id_x() & 63;
    for (int j0 = lo; j0 < hi; j0 += 64) {
      const int n = min(64, hi - j0), j = j0 + min(lane, n - 1);
      const bf16_t *r0 = y0 + (int64_t)j * y0_sr, *r1 = y1 + (int64_t)j * y1_sr;
      float s = nl[KEY ? j : 0], dp = nd[KEY ? j : 0];
      for (int e = 0; e < D; e++) {
        s = fmaf((float)x0[e], (float)r0[e], s);
        dp = fmaf((float)x1[e], (float)r1[e], dp);
      }
      const float pr = fast_exp2(s * c), ds = pr * dp;
      for (int i = 0; i < n; i++) {
        const float wd = __shfl(ds, i, 64), wp = __shfl(pr, i, 64);
#pragma unroll
        for (int e = 0; e < D / 64; e++) {
          a0[e] = fmaf(wd, (float)y0[(int64_t)(j0 + i) * y0_sr + e * 64 + lane], a0[e]);
          if constexpr (KEY) a1[e] = fmaf(wp, (float)y1[(int64_t)(j0 + i) * y1_sr + e * 64 + lane], a1[e]);
        }
      }
    }
  }
  __device__ __forceinline__ void store(const float* a, float factor, bf16_t* to) const {
    const int lane = __builtin_amdgcn_workitem_id_x() & 63;
#pragma unroll
    for (int e = 0; e < D / 64; e++) to[e * 64 + lane] = (bf16_t)(a[e] * factor);
  }
};

// Four columns of the sum of all shares, `stride` floats from one to the next, to `to` (null: nowhere).  Is one of them not finite?
__device__ __forceinline__ bool join_part(const float* part, int64_t stride, int shares, float factor, bf16_t* to) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < shares; s++) {
    const f32x4 y = *(const f32x4*)(part + s * stride);
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] += y[e];
  }
  if (!to) return false;
  *(u32x2*)to = u32x2{pack_bf16(sum[0] * factor, sum[1] * factor), pack_bf16(sum[2] * factor, sum[3] * factor)};
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad |= not_finite(sum[e]);
  return bad;
}

template <int MT>
__device__ __forceinline__ bool any_not_finite(const f32x16 (&acc)[MT]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) bad |= not_finite(acc[i][e]);
  return bad;
}

template <int MT>
__device__ __forceinline__ void clear(f32x16 (&acc)[MT]) {
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) acc[i][e] = 0.f;
}

__device__ __forceinline__ bf16x8 pack_half(const f32x16& x, int kb) {
  return kb == 0 ? pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]) : pack8(x[8], x[9], x[10], x[11], x[12], x[13], x[14], x[15]);
}

#endif

// keys in three buffers, values in two
template <int D>
constexpr int dq_lds(int waves) {
  const int bufs = 5 * 64 * D * 2, out = waves * 32 * (D * 2 + 16);
  return bufs > out ? bufs : out;
}

#if defined(__HIP_DEVICE_COMPILE__)

// the first of 16 elements in slot g of N: all of them are through their three slots at the end
template <int N>
struct DqSlots {
  static constexpr int lo(int g) { return g <= 0 ? 0 : g >= N - 2 ? 16 : g * 16 / (N - 2); }
};

#endif

// ---- dq: 32 query rows per wave, steps of 32 keys.  S^T and dP^T = V do^T with the rows of q and do as B operands in registers, so a lane
// owns a query column, and dS^T is in the B operand's layout of dq^T += K^T dS^T as it is.  A step forms S and dP of the coming 32 keys on the
// matrix cores while the vector ALU turns those of the present ones into dS, and adds them.  The barrier of a tile of 64 keys lies between its
// two steps' products: the first S of the next tile is formed beside the second dS of this one, whose keys stay (hence three buffers).
//
// delta comes from o, which is rounded: sum_j P (dP - delta), which should be 0, is off.  In rows of few keys, where o is no mean of many values, that is as
// large as the rounding of dS; waves whose rows have all their keys in one tile form that sum first and take it off (settle): dq and dk of the sequences
// below are then off by 0.0024 of their size instead of 0.0025 (0.0024 instead of 0.0026 if they have 110 tokens each), for 1 % of the time.
//
// 12 sequences of up to 2047 tokens, 32 heads over 8 of 128, causal: 244 us with a step's products, vector work and sums one behind the other, 228 so,
// 222 without tiles that none of a wave's rows sees, 225 with settled deltas (224 to 232 from card to card: 770 to 800 TFLOP/s), matrix cores busy 48 % of the
// cycles.  16384 rows of 16 heads of 64 over 811 keys in
// four texts: 46 -> 44 us. ----

template <int D, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void packed_dq_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = PackedLds<D>;
  using P = PackedOperands<D>;
  constexpr int KS = D / 16, MTD = D / 32, TILE = S::TILE;
  const int per = SPLIT ? p.H * p.shares : p.H;
  const int id = __builtin_amdgcn_workgroup_id_x(), place = id / per, j = id - place * per, share = SPLIT ? j / p.H : 0;
  PackedTile w;
  if (!find_tile<NW * 32>(p.q_off, p.T, p.k_off, p.Tk, p.B, p.slots - 1 - place, false, w)) return;
  const int h = packed_head(j - share * p.H, p.H), hk = h / p.G;
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  const int wave = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_workitem_id_x() >> 6);
  const int hh = lane >> 5, r = lane & 31;
  const S at(lane);
  const int m_all = w.other_n;
  const int q0 = w.row0 + wave * 32, shift = p.causal ? m_all - w.n : m_all;
  auto all_seen_by = [&](int row) { return max(0, p.causal ? min(m_all, row + shift + 1) : m_all); };
  const int T_all = (all_seen_by(min(w.row0 + NW * 32, w.n) - 1) + 63) >> 6;
  const Share part = SPLIT ? share_of(T_all, share, p.shares) : Share{0, T_all};
  // from here on keys are those of the share
  const int T = part.T, k_first = w.other_first + 64 * part.t0, m = SPLIT ? max(0, min(m_all - 64 * part.t0, 64 * T)) : m_all;
  auto seen_by = [&](int row) { return SPLIT ? max(0, min(m, all_seen_by(row) - 64 * part.t0)) : all_seen_by(row); };
  const int row = min(q0 + r, w.n - 1);
  const int seen = seen_by(row), seen_first = __builtin_amdgcn_readfirstlane(seen);
  const bool live = q0 + r < w.n;
  const int64_t trow = w.first + row;
  const float c = p.c;

  // the first tile is requested ahead of the rows, so that one latency covers both
  const bf16_t *kp = p.k + hk * p.k_sh + (int64_t)k_first * p.k_sr, *vp = p.v + hk * p.v_sh + (int64_t)k_first * p.v_sr;
  const int k_srb = (int)p.k_sr * 2, v_srb = (int)p.v_sr * 2;
  const i32x4 krsrc = packed_rsrc(kp, m, S::ROWB, k_srb), vrsrc = packed_rsrc(vp, m, S::ROWB, v_srb);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LVAR_LDS char*)smem;
  auto request = [&](int t, int k_pl) {   // tile t into the place k_pl of the keys' ring
    fill_tile<D, NW>(krsrc, k_srb, 64 * t, lds0 + k_pl, wave, lane);
    fill_tile<D, NW>(vrsrc, v_srb, 64 * t, lds0 + (3 + (t & 1)) * TILE, wave, lane);
  };
  // without dq: only statistics, and deltas that are settled (beyond three tiles no wave has one alone)
  const bool settle = !SPLIT && p.settle, runs = p.dq || (settle && T <= 3);
  if (runs && T > 0) request(0, 0);

  // q and do of the row; delta from do and o, half of the columns in each of the lanes l and l^32
  bf16x8 qf[KS], gf[KS];
  float delta = 0.f;
  {
    const bf16_t *qp = p.q + h * p.q_sh + trow * p.q_sr + hh * 8, *gp = p.g + h * p.g_sh + trow * p.g_sr + hh * 8, *op = p.o + h * p.o_sh + trow * p.o_sr + hh * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      qf[ks] = *(const bf16x8*)(qp + ks * 16);
      gf[ks] = *(const bf16x8*)(gp + ks * 16);
      const bf16x8 of = *(const bf16x8*)(op + ks * 16);
#pragma unroll
      for (int e = 0; e < 8; e++) delta = fmaf((float)gf[ks][e], (float)of[e], delta);
    }
  }
  delta = xhalf_sum(delta);
  const int64_t stat = (int64_t)h * p.T + trow;
  const float M = p.M[stat], L = p.L[stat];
  // (no key, or none with a weight: M and L as the forward pass writes them then; with M in the start of its sums P would be NaN)
  const bool sees = all_seen_by(row) > 0 && !(bits_of(M) == 0xff800000u && bits_of(L) == 0x3f800000u);
  const float nl = sees ? -(M + __builtin_amdgcn_logf(L)) / c : -INFINITY;
  float nd = sees ? -delta : 0.f;
  if (hh == 0 && live && share == 0) {
    float* to = p.stats + (int64_t)h * 2 * p.T + trow;
    to[0] = nl;
    to[p.T] = nd;
  }

  f32x16 acc[MTD];
  clear(acc);
  if (!runs) return;
  if (T > 0) {
    const uint32_t k_rows = lds0 + at.row_at, v_rows = k_rows + 3 * TILE, k_cols = lds0 + at.tr_at;
    constexpr int NS = 2 * KS, NP = 2 * MTD, NT = NS + NP, AHEAD = 2;
    auto land = [&]() {
      wait_fills<0>();
      __syncthreads();
    };
    // starting values of S and dP; -infinity for keys that a row does not see
    auto starts = [&](auto masked, int t, int sub, f32x16& s, f32x16& dp) {
      const int lim = seen - 64 * t - 32 * sub - 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        s[i] = decltype(masked)::value && 8 * (i >> 2) + (i & 3) >= lim ? -INFINITY : nl;
        dp[i] = nd;
      }
    };
    // FIRST: S and dP of 32 keys, rows at `kr` and `vr`, in ns and ndp.  SECOND: those in s and dp are turned into dS and added, keys at `kc`.
    auto step = [&](auto first, auto second, uint32_t kr, uint32_t vr, uint32_t kc, f32x16& s, f32x16& dp, f32x16& ns, f32x16& ndp) {
      constexpr bool FIRST = decltype(first)::value, SECOND = decltype(second)::value;
      bf16x8 frag[NT];
      uint32_t pw[8];
      auto operand = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < NS) { if constexpr (FIRST) frag[i] = P::rows(i & 1 ? vr : kr, i >> 1); }
        else if constexpr (i < NT) { if constexpr (SECOND) frag[i] = P::columns(kc, (i - NS) / MTD, (i - NS) % MTD); }
      };
      using Sch = DqSlots<NS>;
      auto slot = [&](auto gc) {
        constexpr int g = decltype(gc)::value;
        if constexpr (SECOND) {
          static_for<Sch::lo(g - 2), Sch::lo(g - 1)>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            s[e] *= dp[e];
            if constexpr (e & 1) pw[e >> 1] = pack_bf16(s[e - 1], s[e]);
          });
          static_for<Sch::lo(g - 1), Sch::lo(g)>([&](auto ec) { constexpr int e = decltype(ec)::value; s[e] = fast_exp2(s[e]); });
          static_for<Sch::lo(g), Sch::lo(g + 1)>([&](auto ec) { constexpr int e = decltype(ec)::value; s[e] *= c; });
        }
      };
      static_for<FIRST ? 0 : NS, (FIRST ? 0 : NS) + AHEAD>(operand);
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, NS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (FIRST) {
          operand(std::integral_constant<int, i + AHEAD>{});
          if constexpr (i & 1) ndp = mfma32(frag[i], gf[i >> 1], ndp); else ns = mfma32(frag[i], qf[i >> 1], ns);
        }
        slot(ic);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (SECOND) {
        slot(std::integral_constant<int, NS>{});
        static_for<NS, NT>([&](auto ic) {
          constexpr int i = decltype(ic)::value, kb = (i - NS) / MTD, x = (i - NS) % MTD;
          operand(std::integral_constant<int, i + AHEAD>{});
          acc[x] = mfma32(frag[i], __builtin_bit_cast(bf16x8, u32x4{pw[4 * kb], pw[4 * kb + 1], pw[4 * kb + 2], pw[4 * kb + 3]}), acc[x]);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    };
    using Yes = std::true_type;
    using No = std::false_type;
    constexpr int SUB_ROWS = 32 * S::ROWB, SUB_COLS = 32 * S::ROWB;
    f32x16 sa, da, sb, db;
    int k_pl = 0, k_next = TILE;   // places of the present tile and of the next one
    land();
    if (T > 1) request(1, TILE);
    auto arrive = [&](int t) {   // tile t is there, the next one is requested
      land();
      k_pl = k_next;
      k_next = k_pl == 2 * TILE ? 0 : k_pl + TILE;
      if (t + 1 < T) request(t + 1, k_next);
    };
    auto round = [&](int t, auto masked) {   // the second step of tile t - 1, and the first of tile t
      const int k_last = k_pl;
      arrive(t);
      const uint32_t vr = v_rows + (t & 1) * TILE;
      starts(masked, t, 0, sa, da);
      step(Yes{}, Yes{}, k_rows + k_pl, vr, k_cols + k_last + SUB_COLS, sb, db, sa, da);
      starts(masked, t, 1, sb, db);
      step(Yes{}, Yes{}, k_rows + k_pl + SUB_ROWS, vr + SUB_ROWS, k_cols + k_pl, sa, da, sb, db);
    };
    const int mine = q0 < w.n ? (seen_by(min(q0 + 32, w.n) - 1) + 63) >> 6 : 0;   // tiles that a row of the wave sees
    const int whole = min(mine, seen_first >> 6);                                 // and that all of them see whole
    int t = 1;
    if (mine > 0) {
      if (settle && mine == 1) {
        starts(Yes{}, 0, 0, sa, da);
        step(Yes{}, No{}, k_rows, v_rows, k_cols, sb, db, sa, da);
        starts(Yes{}, 0, 1, sb, db);
        step(Yes{}, No{}, k_rows + SUB_ROWS, v_rows + SUB_ROWS, k_cols, sa, da, sb, db);
        const int lim = seen - 4 * hh;
        float off = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = 8 * (i >> 2) + (i & 3);
          const float x = fast_exp2(sa[i] * c) * da[i], y = fast_exp2(sb[i] * c) * db[i];
          off += (key < lim ? x : 0.f) + (key + 32 < lim ? y : 0.f);
        }
        nd -= xhalf_sum(off);
        if (hh == 0 && live) p.stats[(int64_t)h * 2 * p.T + p.T + trow] = nd;
      }
      starts(Yes{}, 0, 0, sa, da);
      step(Yes{}, No{}, k_rows, v_rows, k_cols, sb, db, sa, da);
      starts(Yes{}, 0, 1, sb, db);
      step(Yes{}, Yes{}, k_rows + SUB_ROWS, v_rows + SUB_ROWS, k_cols, sa, da, sb, db);
      for (; t < whole; t++) round(t, No{});
      for (; t < mine; t++) round(t, Yes{});
      step(No{}, Yes{}, k_rows, v_rows, k_cols + k_pl + SUB_COLS, sb, db, sa, da);
    }
    for (; t < T; t++) arrive(t);
    __syncthreads();
  }
  if constexpr (SPLIT) {   // packed_dq_join_kernel does the rest
    store_part<D>(smem + wave * (32 * (D * 2 + 16)), acc, p.parts + (((int64_t)share * p.H + h) * p.T + w.first + q0) * D, w.n - q0, lane);
    return;
  }
  if (!p.dq) return;
  bf16_t* to = p.dq + h * p.dq_sh + (int64_t)(w.first + q0) * p.dq_sr;
  store_rows<D>(smem + wave * (32 * (D * 2 + 16)), acc, p.scale, to, p.dq_sr, w.n - q0, lane);
  if (p.causal || m_all % 64 != 0) {
    uint64_t rows = __builtin_amdgcn_ballot_w64(any_not_finite(acc) && live);
    rows = (rows | rows >> 32) & 0xffffffffu;
    if (rows) wait_fills<0>();   // the rows as stored above are written again
    while (rows) {
      const int i = __builtin_ctzll(rows);
      rows &= rows - 1;
      const int64_t x = w.first + q0 + i;
      const float nli = __shfl(nl, i, 64), ndi = __shfl(nd, i, 64);
      CarefulRow<D, false> a;
      a.clear();
      a.add(p.q + h * p.q_sh + x * p.q_sr, p.g + h * p.g_sh + x * p.g_sr, kp, p.k_sr, vp, p.v_sr, 0, __shfl(seen, i, 64), &nli, &ndi, c);
      a.store(a.a0, p.scale, to + i * p.dq_sr);
    }
  }
#endif
}

// dq of a launch whose workgroups shared keys, from the parts in their order: a lane per four columns.
template <int D>
__global__ __launch_bounds__(256) void packed_dq_join_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int LPR = D / 4, RPG = 256 / LPR;
  const int tid = __builtin_amdgcn_workitem_id_x(), column = tid % LPR * 4;
  const int64_t rows = (int64_t)p.H * p.T, x = (int64_t)__builtin_amdgcn_workgroup_id_x() * RPG + tid / LPR, at = min(x, rows - 1);
  const int h = (int)(at / p.T), row = (int)(at - (int64_t)h * p.T);
  uint64_t left = __builtin_amdgcn_ballot_w64(join_part(p.parts + at * D + column, rows * D, p.shares, p.scale, x < rows ? p.dq + h * p.dq_sh + (int64_t)row * p.dq_sr + column : nullptr));
  if (left) wait_fills<0>();   // the rows as stored above are written again
  while (left) {
    const int i = __builtin_ctzll(left) / LPR * LPR;   // the first lane of a row
    left &= i + LPR < 64 ? ~0ull << (i + LPR) : 0ull;
    const int hi = __builtin_amdgcn_readlane(h, i), ri = __builtin_amdgcn_readlane(row, i), hk = hi / p.G;
    PackedTile w;
    find_row(p.q_off, p.T, p.k_off, p.Tk, p.B, ri, w);
    if (!p.causal && w.other_n % 64 == 0) continue;
    const int seen = p.causal ? max(0, min(w.other_n, w.row0 + w.other_n - w.n + 1)) : w.other_n;
    const float* st = p.stats + (int64_t)hi * 2 * p.T + ri;
    CarefulRow<D, false> a;
    a.clear();
    a.add(p.q + hi * p.q_sh + (int64_t)ri * p.q_sr, p.g + hi * p.g_sh + (int64_t)ri * p.g_sr, p.k + hk * p.k_sh + (int64_t)w.other_first * p.k_sr, p.k_sr,
          p.v + hk * p.v_sh + (int64_t)w.other_first * p.v_sr, p.v_sr, 0, seen, st, st + p.T, p.c);
    a.store(a.a0, p.scale, p.dq + hi * p.dq_sh + (int64_t)ri * p.dq_sr);
  }
#endif
}

// ---- dk and dv: tiles of 128 keys (head_dim 64 and 256: 64) and of 64 query rows (256: 32) of every query head that shares the key head.
//
// Two waves share 32 keys.  One forms S = q k^T and P and adds do^T P to dv^T; the other forms dP = do v^T, takes P from the first through LDS,
// and adds q^T dS to dk^T.  Each has one operand (k or v) and one sum in registers, which leaves room for what hides latency: it forms S or dP
// of the coming tile on the matrix cores while the vector ALU turns those of the present one into P or dS, and then adds the present one to its
// sum.  (One wave with both sums: 2500 cycles per 32 products if it has its SIMD to itself, for it issues an instruction every four cycles at most;
// as two per SIMD without a tile in hand 2000; of these the matrix cores need 1024.)  The second wave is a tile behind the
// first, so that P passes behind the barrier that a tile has anyway.  A lane owns a key column: P and dS are in the B operand's layout
// of the second product as they leave the vector ALU.  S and dP start at -(M + log2 L) / c and -delta of their rows: P is one exp2 of c
// times the sum, dS one product.
//
// Tiles come from the last rows to the first, all heads of a tile behind each other: the workgroups of a sequence, which all end at
// its last rows, read the same tile at about the same time, from the L2 (from the first rows on, 71 % of the reads missed it); half of the reads
// still come from further away, so tiles are requested LEAD rounds ahead.  The same sequences 277 to 289 us from card to card, 825 to 860 TFLOP/s, matrix
// cores busy 50 %. ----

template <int D>
struct Dkv {
  // Pairs of waves.  head_dim 64: two, so that two workgroups share a compute unit and wait at barriers of their own (16384 rows of 16 heads over 725
  // keys 72 -> 54 us); 128: four, half of the reads for the same time (12 sequences of 32 over 8 heads 263 / 254 us); 256: one wave per SIMD.
  static constexpr int KW = D == 128 ? 4 : 2, WAVES = 2 * KW, KEYS = 32 * KW;
  static constexpr int SUB = D == 256 ? 1 : 2, R = 32 * SUB, TILE = R * D * 2;    // 32-row blocks and rows of a tile, its bytes
  // tiles of q: t-1 .. t+1 are in use, of do: t
  static constexpr int LEAD = D == 256 ? 2 : 1, Q_RING = LEAD + 3, G_RING = LEAD + 1;
  static constexpr int G_AT = Q_RING * TILE, P_AT = G_AT + G_RING * TILE, P_WAVE = R * 32 * 3;   // P: [parity][pair], 24 bits each
  static constexpr int STAT_AT = P_AT + 2 * KW * P_WAVE, STAT_WAVE = Q_RING * 256;               // statistics: [wave][place in the ring]
  static constexpr int OUT = WAVES * 32 * (D * 2 + 16);
  static constexpr int bytes() { return STAT_AT + WAVES * STAT_WAVE > OUT ? STAT_AT + WAVES * STAT_WAVE : OUT; }
};

#if defined(__HIP_DEVICE_COMPILE__)

// P passes between two waves as the upper 24 bits of its fp32, cut (less than 2^-15 of it is lost, where dS is rounded to 2^-9): 16 of two elements to a
// word, the next 8 of four to another.  (As bf16 dk is off by 0.0030 of its size instead of 0.0025, as dq; rounded once, at its end, it would be by
// 0.0017.  It costs 5 % of the kernel at head_dim 128, 15 % at 64: 272 -> 286 us, 53 -> 61 us.)
__device__ __forceinline__ uint32_t word(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ uint32_t upper16(float a, float b) { return __builtin_amdgcn_perm(word(b), word(a), 0x07060302u); }
__device__ __forceinline__ uint32_t next8(float a, float b, float c, float d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(word(d), word(c), 0x0c0c0501u), __builtin_amdgcn_perm(word(b), word(a), 0x0c0c0501u), 0x05040100u);
}
// element E of a group of eight
template <int E>
__device__ __forceinline__ float unpack24(uint32_t upper, uint32_t next) {
  return __builtin_bit_cast(float, __builtin_amdgcn_perm(upper, next, (E & 1 ? 0x07060000u : 0x05040000u) | (E & 3) << 8 | 0x0cu));
}

// the first of N elements in slot g: three quarters over the NS steps of the first product, the others over the first HB of the second
template <int N, int NS, int HB>
struct DkvSlots {
  static constexpr int lo(int g) {
    constexpr int early = N * 3 / 4;
    return g <= 0 ? 0 : g < NS ? g * early / NS : g < NS + HB ? early + (g - NS) * (N - early) / HB : N;
  }
};

// dk or dv of one key, see CarefulRow; rows from `from` on see it
template <int D, int ROLE>
__device__ __forceinline__ void careful_key(const PackedParams& p, const PackedTile& w, int hk, int key, int from) {
  const int64_t x = w.first + key;
  CarefulRow<D, true> a;
  a.clear();
  for (int head = 0; head < p.G; head++) {
    const int hq = hk * p.G + head;
    const float* st = p.stats + (int64_t)hq * 2 * p.T + w.other_first;
    a.add(p.k + hk * p.k_sh + x * p.k_sr, p.v + hk * p.v_sh + x * p.v_sr, p.q + hq * p.q_sh + (int64_t)w.other_first * p.q_sr, p.q_sr,
          p.g + hq * p.g_sh + (int64_t)w.other_first * p.g_sr, p.g_sr, min(from, w.other_n), w.other_n, st, st + p.T, p.c);
  }
  if constexpr (ROLE == 0) a.store(a.a1, 1.f, p.dv + hk * p.dv_sh + x * p.dv_sr);
  else a.store(a.a0, p.scale, p.dk + hk * p.dk_sh + x * p.dk_sr);
}

template <int D, int ROLE>   // ROLE 0: dv, 1: dk
__device__ __forceinline__ void dkv_wave(const PackedParams& p, char* smem, const PackedTile& w, const int hk, const int share, const int all_waves) {
  using S = PackedLds<D>;
  using Q = Dkv<D>;
  using P = PackedOperands<D>;
  constexpr int KS = D / 16, MTD = D / 32, TILE = Q::TILE, SUB = Q::SUB, NE = 16 * SUB;
  const int lane = __builtin_amdgcn_workitem_id_x() & 63, hh = lane >> 5, r = lane & 31;
  const int wave = all_waves & (Q::KW - 1);
  const S at(lane);
  const int q_first = w.other_first, n = w.other_n;
  const int k0 = w.row0 + wave * 32, key = min(k0 + r, w.n - 1);
  const int shift = w.n - n;
  const int from = p.causal ? max(0, key - shift) : 0;   // the first row that sees the lane's key
  const int b0 = p.causal ? min(max(0, w.row0 - shift), n) / Q::R : 0, last = (n + Q::R - 1) / Q::R - 1;
  // tiles of this workgroup's share: T_all * share / shares ..
  const int64_t T_all = (int64_t)max(0, last + 1 - b0) * p.G;
  const int t_first = (int)(T_all * share / p.shares), T = (int)(T_all * (share + 1) / p.shares) - t_first;
  const int blk_first = last - t_first / p.G, head_first = t_first % p.G;
  const int whole0 = p.causal ? max(0, k0 + 31 - shift) : 0;   // rows from here on see all keys of the wave
  // those that see a key of this pair of waves: none of the last ones, if causal
  const int b0_mine = p.causal ? min(max(0, k0 - shift), n) / Q::R : 0;
  const int64_t T_mine = k0 < w.n ? (int64_t)max(0, last + 1 - b0_mine) * p.G - t_first : 0;
  const int mine = __builtin_amdgcn_readfirstlane((int)max((int64_t)0, min(T_mine, (int64_t)T)));
  const float c = p.c;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LVAR_LDS char*)smem;

  f32x16 acc[MTD];
  clear(acc);
  if (T > 0) {
    // The first waves of the pairs request q, the others do, each with its own copy of the statistic that its sums start at.
    constexpr int RING = ROLE ? Q::G_RING : Q::Q_RING, FILLS = Q::R / S::RPI / Q::KW + 1;
    const int srb = (int)(ROLE ? p.g_sr : p.q_sr) * 2, bytes = __builtin_amdgcn_readfirstlane((n - 1) * srb + S::ROWB);
    const int64_t head_stride = ROLE ? p.g_sh : p.q_sh;
    const bf16_t* const x0 = (ROLE ? p.g + hk * p.G * p.g_sh : p.q + hk * p.G * p.q_sh) + (int64_t)q_first * (ROLE ? p.g_sr : p.q_sr);
    const float* const s0 = p.stats + ((int64_t)hk * p.G * 2 + ROLE) * p.T + q_first;
    const uint32_t fill0 = lds0 + (ROLE ? Q::G_AT : 0), stat0 = lds0 + Q::STAT_AT + all_waves * Q::STAT_WAVE;
    auto after = [](int pl, int ring) { return pl + TILE == ring * TILE ? 0 : pl + TILE; };   // the next place of a ring
    int f_t = 0, f_blk = blk_first, f_head = head_first, f_pl = 0;   // the tile that is requested next
    const bf16_t* xp = x0 + head_first * head_stride;
    const float* sp = s0 + 2 * (int64_t)head_first * p.T;
    auto request = [&]() {
      const bool there = f_t < T;                    // behind the last tile: as many fills, of nothing
      const int row = there ? f_blk * Q::R : 0;
      fill_rows<D, Q::KW, Q::R>(packed_rsrc(xp, there ? bytes : 0), srb, row, fill0 + f_pl, wave, lane);
      const i32x4 rsrc = packed_rsrc(sp, there ? n * 4 : 0);
      const int voff = lane * 4, soff = row * 4;
      const uint32_t m0v = stat0 + f_pl / (TILE / 256);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(m0v), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
      f_t++;
      f_pl = after(f_pl, RING);
      const bool wrap = ++f_head == p.G;
      f_head = wrap ? 0 : f_head;
      f_blk -= wrap ? 1 : 0;
      xp = wrap ? x0 : xp + head_stride;
      sp = wrap ? s0 : sp + 2 * (int64_t)p.T;
    };
    // Rows behind the last one, in the first tile of every head, have read zeros as their statistics: they see nothing.
    auto patch = [&](int t, int pl) {
      if (t_first + t < p.G && last * Q::R + lane >= n) *(LVAR_LDS float*)(uintptr_t)(stat0 + pl / (TILE / 256) + lane * 4) = ROLE ? 0.f : -INFINITY;
    };

    constexpr int AHEAD_T = Q::LEAD + (ROLE ? 0 : 1);   // tiles requested ahead of the first round
    for (int x = 0; x < AHEAD_T; x++) request();
    bf16x8 xf[KS];   // rows of k or of v
    {
      const bf16_t* kv = ROLE ? p.v + hk * p.v_sh + (int64_t)(w.first + key) * p.v_sr : p.k + hk * p.k_sh + (int64_t)(w.first + key) * p.k_sr;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) xf[ks] = *(const bf16x8*)(kv + hh * 8 + ks * 16);
    }
    const uint32_t row_at = fill0 + at.row_at, col_at = lds0 + (ROLE ? 0 : Q::G_AT) + at.tr_at;
    const uint32_t p_at = lds0 + Q::P_AT + wave * Q::P_WAVE + lane * 16;
    constexpr int NS = SUB * KS, NP = 2 * SUB * MTD, NT = NS + NP, AHEAD = READ_AHEAD;
    // places of the tile whose S or dP is formed (rows) and of the one that is added (columns)
    int r_pl = 0, c_pl = 0, r_blk = blk_first, r_head = head_first;
    // starting values of S or dP of the tile at r_pl; -infinity where a row does not see the lane's key
    auto starts = [&](f32x16 (&s)[SUB]) {
      LVAR_LDS const float* st = (LVAR_LDS const float*)(uintptr_t)(stat0 + r_pl / (TILE / 256));
#pragma unroll
      for (int b = 0; b < SUB; b++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
          const f32x4 v = *(LVAR_LDS const f32x4*)(st + 32 * b + 8 * a + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; e++) s[b][4 * a + e] = v[e];
        }
      if constexpr (ROLE == 0) {
        if (r_blk * Q::R < whole0) {
          const int lo = from - r_blk * Q::R - 4 * hh;
#pragma unroll
          for (int b = 0; b < SUB; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[b][e] = 32 * b + 8 * (e >> 2) + (e & 3) >= lo ? s[b][e] : -INFINITY;
        }
      }
    };
    auto next_rows = [&]() {
      r_pl = after(r_pl, RING);
      const bool wrap = ++r_head == p.G;
      r_head = wrap ? 0 : r_head;
      r_blk -= wrap ? 1 : 0;
    };
    int landed = 0, l_pl = 0;   // tiles that have landed
    auto settle = [&](auto rounds) {   // all but the last `rounds` requested tiles have
      wait_fills<decltype(rounds)::value * FILLS>();
      patch(landed, l_pl);
      landed++;
      l_pl = after(l_pl, RING);
      __syncthreads();
    };
    // A round.  Tile t of this wave: its S or dP is in s.  FIRST: that of the coming tile is formed, in nx; SECOND: tile t is added to the sum.
    auto round = [&](int t, auto first, auto second, f32x16 (&s)[SUB], f32x16 (&nx)[SUB]) {
      constexpr bool FIRST = decltype(first)::value, SECOND = decltype(second)::value;
      const uint32_t rows = row_at + r_pl, cols = col_at + c_pl, pt = p_at + (t & 1) * Q::KW * Q::P_WAVE;
      const uint32_t pt8 = pt + Q::R * 64 - lane * 8;
      bf16x8 frag[NT];
      uint32_t pw[8 * SUB];   // P or dS, packed
      uint32_t up[4], lo[2];  // P for the other wave
      u32x4 pin[2 * SUB];     // and from it
      u32x2 pin8[2 * SUB];
      auto operand = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (i < NS) { if constexpr (FIRST) frag[i] = P::rows(rows + i % SUB * 32 * S::ROWB, i / SUB); }
        else if constexpr (i < NT) { if constexpr (SECOND) frag[i] = P::columns(cols, (i - NS) / MTD, (i - NS) % MTD); }
      };
      using Sch = DkvSlots<NE, NS, SUB == 1 ? NP / 4 : NP / 2>;
      // (what a product takes is finished two slots ahead of it)
      static_assert(Sch::lo(NS - 2) >= 8 && Sch::lo(NS + MTD - 2) >= 16 && (SUB == 1 || (Sch::lo(NS + 2 * MTD - 2) >= 24 && Sch::lo(NS + 3 * MTD - 2) >= 32)));
      auto finish = [&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (ROLE == 1) s[e / 16][e % 16] *= unpack24<e % 8>(pin[e / 8][e % 8 / 2], pin8[e / 8][e % 8 / 4]);
        if constexpr (e & 1) pw[e >> 1] = pack_bf16(s[e / 16][e % 16 - 1], s[e / 16][e % 16]);
        if constexpr (ROLE == 0 && e % 2 == 1) up[e % 8 / 2] = upper16(s[e / 16][e % 16 - 1], s[e / 16][e % 16]);
        if constexpr (ROLE == 0 && e % 4 == 3) lo[e % 8 / 4] = next8(s[e / 16][e % 16 - 3], s[e / 16][e % 16 - 2], s[e / 16][e % 16 - 1], s[e / 16][e % 16]);
        if constexpr (ROLE == 0 && e % 8 == 7) {
          *(LVAR_LDS u32x4*)(uintptr_t)(pt + e / 8 * 1024) = u32x4{up[0], up[1], up[2], up[3]};
          *(LVAR_LDS u32x2*)(uintptr_t)(pt8 + e / 8 * 512) = u32x2{lo[0], lo[1]};
        }
      };
      auto slot = [&](auto gc) {
        constexpr int g = decltype(gc)::value;
        if constexpr (SECOND) {
          static_for<Sch::lo(g - 2), Sch::lo(g - 1)>(finish);
          if constexpr (ROLE == 0) {
            static_for<Sch::lo(g - 1), Sch::lo(g)>([&](auto ec) { constexpr int e = decltype(ec)::value; s[e / 16][e % 16] = fast_exp2(s[e / 16][e % 16]); });
            static_for<Sch::lo(g), Sch::lo(g + 1)>([&](auto ec) { constexpr int e = decltype(ec)::value; s[e / 16][e % 16] *= c; });
          }
        }
      };
      if constexpr (ROLE == 1 && SECOND) {
#pragma unroll
        for (int i = 0; i < 2 * SUB; i++) {
          pin[i] = *(LVAR_LDS const u32x4*)(uintptr_t)(pt + i * 1024);
          pin8[i] = *(LVAR_LDS const u32x2*)(uintptr_t)(pt8 + i * 512);
        }
      }
      if constexpr (FIRST) starts(nx);
      static_for<FIRST ? 0 : NS, (FIRST ? 0 : NS) + AHEAD>(operand);
      request();
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, NS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (FIRST) {
          operand(std::integral_constant<int, i + AHEAD>{});
          nx[i % SUB] = mfma32(frag[i], xf[i / SUB], nx[i % SUB]);
        }
        slot(ic);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (SECOND) {
        static_for<NS, NT>([&](auto ic) {
          constexpr int i = decltype(ic)::value, kb = (i - NS) / MTD, m = (i - NS) % MTD;
          operand(std::integral_constant<int, i + AHEAD>{});
          acc[m] = mfma32(frag[i], __builtin_bit_cast(bf16x8, u32x4{pw[4 * kb], pw[4 * kb + 1], pw[4 * kb + 2], pw[4 * kb + 3]}), acc[m]);
          slot(ic);
          __builtin_amdgcn_sched_barrier(0);
        });
        c_pl = after(c_pl, ROLE ? Q::Q_RING : Q::G_RING);
      }
      if constexpr (FIRST) next_rows();
      settle(std::integral_constant<int, Q::LEAD - 1>{});
    };
    using Yes = std::true_type;
    using No = std::false_type;
    f32x16 sa[SUB], sb[SUB];
    // ahead of the first round: S(0) by the first waves
    settle(std::integral_constant<int, AHEAD_T - 1>{});
    if constexpr (ROLE == 0) {
      starts(sa);
      static_for<0, NS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        sa[i % SUB] = mfma32(P::rows(row_at + i % SUB * 32 * S::ROWB, i / SUB), xf[i / SUB], sa[i % SUB]);
      });
      next_rows();
      settle(std::integral_constant<int, Q::LEAD - 1>{});
    } else {
      __syncthreads();
      round(-1, Yes{}, No{}, sb, sa);   // the first round forms dP(0)
    }
    int t = 0;
    for (; t + 2 < mine; t += 2) {
      round(t, Yes{}, Yes{}, sa, sb);
      round(t + 1, Yes{}, Yes{}, sb, sa);
    }
    if (t + 1 < mine) {
      round(t, Yes{}, Yes{}, sa, sb);
      round(t + 1, No{}, Yes{}, sb, sa);
    } else if (mine > 0) {
      round(t, No{}, Yes{}, sa, sb);
    }
    for (t = mine; t < T; t++) {
      request();
      settle(std::integral_constant<int, Q::LEAD - 1>{});
    }
    if constexpr (ROLE == 0) __syncthreads();   // the others' last round
    wait_fills<0>();
    __syncthreads();
  }
  bf16_t* out = ROLE ? p.dk : p.dv;
  if (!out) return;
  if (p.shares > 1) {   // as it is, transposed: packed_dkv_join_kernel does the rest
    float* part = p.parts + ((((int64_t)share * 2 + ROLE) * p.Hkv + hk) * p.Tk + w.first + k0 + r) * D + 4 * hh;
    if (k0 + r < w.n) {   // (through LDS, as rows of dq, this spills at head_dim 256)
#pragma unroll
      for (int m = 0; m < MTD; m++)
#pragma unroll
        for (int a = 0; a < 4; a++) *(f32x4*)(part + 32 * m + 8 * a) = f32x4{acc[m][4 * a], acc[m][4 * a + 1], acc[m][4 * a + 2], acc[m][4 * a + 3]};
    }
    return;
  }
  const int64_t out_sr = ROLE ? p.dk_sr : p.dv_sr;
  bf16_t* to = out + hk * (ROLE ? p.dk_sh : p.dv_sh) + (int64_t)(w.first + k0) * out_sr;
  store_rows<D>(smem + all_waves * (32 * (D * 2 + 16)), acc, ROLE ? p.scale : 1.f, to, out_sr, w.n - k0, lane);
  if (p.causal || n % Q::R != 0) {
    uint64_t keys = __builtin_amdgcn_ballot_w64(any_not_finite(acc) && k0 + r < w.n);
    keys = (keys | keys >> 32) & 0xffffffffu;
    if (keys) wait_fills<0>();   // the rows as stored above are written again
    while (keys) {
      const int i = __builtin_ctzll(keys);
      keys &= keys - 1;
      careful_key<D, ROLE>(p, w, hk, k0 + i, __shfl(from, i, 64));
    }
  }
}

#endif

template <int D>
__global__ __launch_bounds__(Dkv<D>::WAVES * 64, D <= 128 ? 2 : 1) void packed_dkv_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int id = __builtin_amdgcn_workgroup_id_x(), place = id / (p.Hkv * p.shares), j = id - place * p.Hkv * p.shares, hk = j % p.Hkv, share = j / p.Hkv;
  PackedTile w;
  if (!find_tile<Dkv<D>::KEYS>(p.k_off, p.Tk, p.q_off, p.T, p.B, place, p.causal, w)) return;
  const int wave = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_workitem_id_x() >> 6);
  if (wave < Dkv<D>::KW) dkv_wave<D, 0>(p, smem, w, hk, share, wave);
  else dkv_wave<D, 1>(p, smem, w, hk, share, wave);
#endif
}

// dk and dv from the sums of the shares of a launch, in their order: a lane per four columns.
template <int D>
__global__ __launch_bounds__(256) void packed_dkv_join_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int LPR = D / 4, RPG = 256 / LPR;
  const int tid = __builtin_amdgcn_workitem_id_x(), column = tid % LPR * 4, role = __builtin_amdgcn_workgroup_id_y();
  bf16_t* out = role ? p.dk : p.dv;
  if (!out) return;
  const int64_t rows = (int64_t)p.Hkv * p.Tk, x = (int64_t)__builtin_amdgcn_workgroup_id_x() * RPG + tid / LPR, at = min(x, rows - 1);
  const int hk = (int)(at / p.Tk), row = (int)(at - (int64_t)hk * p.Tk);
  bf16_t* to = out + hk * (role ? p.dk_sh : p.dv_sh) + (int64_t)row * (role ? p.dk_sr : p.dv_sr) + column;
  uint64_t left = __builtin_amdgcn_ballot_w64(join_part(p.parts + (role * rows + at) * D + column, 2 * rows * D, p.shares, role ? p.scale : 1.f, x < rows ? to : nullptr));
  if (left) wait_fills<0>();   // the rows as stored above are written again
  while (left) {
    const int i = __builtin_ctzll(left) / LPR * LPR;   // the first lane of a row
    left &= i + LPR < 64 ? ~0ull << (i + LPR) : 0ull;
    const int hi = __builtin_amdgcn_readlane(hk, i), ri = __builtin_amdgcn_readlane(row, i);
    PackedTile w;
    find_row(p.k_off, p.Tk, p.q_off, p.T, p.B, ri, w);
    if (!p.causal && w.other_n % Dkv<D>::R == 0) continue;
    const int from = p.causal ? max(0, w.row0 - (w.n - w.other_n)) : 0;
    if (role) careful_key<D, 1>(p, w, hi, w.row0, from); else careful_key<D, 0>(p, w, hi, w.row0, from);
  }
#endif
}

// Workgroups that share the query rows of a key tile, where the key tiles alone leave compute units idle (few keys under many rows, or one key
// head under many query heads): as many as give each unit one (head_dim 64, where it holds two: two), twice that if causal, where the first tile has twice the work of the mean one;
// none gets fewer than SHARE_TILES tiles of an average sequence.  Against one workgroup per tile, the sum of the parts included: 4096 rows of
// 8 heads over one key head of 128, causal 697 -> 102 us (half as many shares 133); of 256 976 -> 192 us; two of 2048 of 8 over 2 heads of 64
// 90 -> 46 us (one a unit: 53); 16384 rows of 16 heads of 128 over 77 keys 353 -> 52 us, of 64 over 811 in four texts 62 -> 57 us.
template <int D>
static int dkv_shares(const PackedParams& p) {
  constexpr int SHARE_TILES = 8;
  const int64_t groups = ((int64_t)p.Tk / Dkv<D>::KEYS + p.B) * p.Hkv, cus = device_cus(), tiles = (int64_t)p.T / p.B * p.G / Dkv<D>::R / (p.causal ? 2 : 1);
  const int64_t most = tiles / SHARE_TILES, want = (p.causal ? 2 : 1) * (D == 64 ? 2 : 1) * cus / (groups > 0 ? groups : 1);
  const int64_t n = want < most ? want : most;
  return n < 2 ? 1 : n > 64 ? 64 : (int)n;
}

template <int D, bool SPLIT>
static int launch_dq(PackedParams p, hipStream_t s) {
  constexpr int NW = 4, LDS = dq_lds<D>(NW);
  p.slots = (int)packed_slots(p.T, p.B, NW * 32);
  const int64_t groups = (int64_t)p.slots * p.H * p.shares, joins = ((int64_t)p.H * p.T * (D / 4) + 255) / 256;
  if (groups * (NW * 64) > 0xffffffffll || (SPLIT && joins * 256 > 0xffffffffll)) return LVAR_EINVAL;
  auto kern = packed_dq_kernel<D, NW, SPLIT>;
  static std::atomic<uint64_t> ready{0};
  if (!ensure_lds_limit((const void*)kern, LDS, ready)) return LVAR_ELAUNCH;
  hipLaunchKernelGGL(kern, dim3((uint32_t)groups), dim3(NW * 64), LDS, s, p);
  if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (SPLIT && joins > 0) hipLaunchKernelGGL(packed_dq_join_kernel<D>, dim3((uint32_t)joins), dim3(256), 0, s, p);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

template <int D>
static int launch_dkv(PackedParams p, hipStream_t s) {
  constexpr int LDS = Dkv<D>::bytes();
  const int64_t groups = packed_slots(p.Tk, p.B, Dkv<D>::KEYS) * p.Hkv * p.shares, joins = ((int64_t)p.Hkv * p.Tk * (D / 4) + 255) / 256;
  if (groups * (Dkv<D>::WAVES * 64) > 0xffffffffll || (p.shares > 1 && joins * 256 > 0xffffffffll)) return LVAR_EINVAL;
  auto kern = packed_dkv_kernel<D>;
  static std::atomic<uint64_t> ready{0};
  if (!ensure_lds_limit((const void*)kern, LDS, ready)) return LVAR_ELAUNCH;
  hipLaunchKernelGGL(kern, dim3((uint32_t)groups), dim3(Dkv<D>::WAVES * 64), LDS, s, p);
  if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (p.shares > 1 && joins > 0) hipLaunchKernelGGL(packed_dkv_join_kernel<D>, dim3((uint32_t)joins, 2), dim3(256), 0, s, p);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

// dq needs no shares where only its statistics are wanted
static int dq_shares(const PackedParams& p, int head_dim, bool wanted) { return wanted ? query_shares(p, head_dim <= 128 ? 2 : 1) : 1; }

template <int D>
static int launch_bwd(PackedParams p, void* workspace, hipStream_t s) {
  p.stats = (float*)workspace;
  p.parts = p.stats + ((int64_t)p.H * 2 * p.T + 3) / 4 * 4;
  p.settle = dq_shares(p, D, true) == 1;
  p.shares = dq_shares(p, D, p.dq != nullptr);
  const int st = p.shares > 1 ? launch_dq<D, true>(p, s) : launch_dq<D, false>(p, s);
  if (st != LVAR_OK || (!p.dk && !p.dv)) return st;
  p.shares = dkv_shares<D>(p);
  return launch_dkv<D>(p, s);
}

// statistics of the rows, and the sums of shares, of dq first and then of dk and dv
int64_t packed_bwd_bytes(const PackedParams& p, int head_dim) {
  const int q = dq_shares(p, head_dim, true), k = head_dim == 64 ? dkv_shares<64>(p) : head_dim == 128 ? dkv_shares<128>(p) : dkv_shares<256>(p);
  const int64_t of_q = q > 1 ? (int64_t)q * p.H * p.T * head_dim : 0, of_k = k > 1 ? (int64_t)k * 2 * p.Hkv * p.Tk * head_dim : 0;
  return 4 * (((int64_t)p.H * 2 * p.T + 3) / 4 * 4 + (of_q > of_k ? of_q : of_k));
}

int launch_packed_bwd(PackedParams p, void* workspace, int head_dim, hipStream_t s) {
  if (head_dim == 128) return launch_bwd<128>(p, workspace, s);
  if (head_dim == 64) return launch_bwd<64>(p, workspace, s);
  if (head_dim == 256) return launch_bwd<256>(p, workspace, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
