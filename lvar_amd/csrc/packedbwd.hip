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

// One row of a gradient whose sums are not finite, pair by pair: 0 * infinity from a row that does not see a key must not stay in it.
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
  // columns lo .. hi-1
  __device__ __forceinline__ void store(const float* a, float factor, bf16_t* to, int lo, int hi) const {
    const int lane = __builtin_amdgcn_workitem_id_x() & 63;
#pragma unroll
    for (int e = 0; e < D / 64; e++)
      if (e * 64 >= lo && e * 64 < hi) to[e * 64 + lane] = (bf16_t)(a[e] * factor);
  }
};

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

template <int D>
constexpr int bwd_lds(int waves, int extra) {
  const int bufs = 4 * 64 * D * 2, out = waves * 32 * (D * 2 + 16);
  return (bufs > out ? bufs : out) + extra;
}

// ---- dq: 32 query rows per wave, tiles of 64 keys.  S^T and dP^T = V do^T with the rows of q and do as B operands in registers, so a lane
// owns a query column, and dS^T is in the B operand's layout of dq^T += K^T dS^T as it is. ----

template <int D, int NW>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void packed_dq_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = PackedLds<D>;
  constexpr int KS = D / 16, MTD = D / 32, TILE = S::TILE;
  const int id = __builtin_amdgcn_workgroup_id_x(), place = id / p.H;
  PackedTile w;
  if (!find_tile<NW * 32>(p.q_off, p.B, p.T, p.slots - 1 - place, w)) return;
  const int h = packed_head(id - place * p.H, p.H), hk = h / p.G;
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  const int wave = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_workitem_id_x() >> 6);
  const int hh = lane >> 5, r = lane & 31;
  const S at(lane);
  int k_first, m;
  packed_range(p.k_off, w.b, p.Tk, k_first, m);
  const int q0 = w.row0 + wave * 32, shift = p.causal ? m - w.n : m;
  auto seen_by = [&](int row) { return max(0, p.causal ? min(m, row + shift + 1) : m); };
  const int T = (seen_by(min(w.row0 + NW * 32, w.n) - 1) + 63) >> 6;
  const int row = min(q0 + r, w.n - 1);
  const int seen = seen_by(row), seen_first = __builtin_amdgcn_readfirstlane(seen);
  const bool live = q0 + r < w.n;
  const int64_t trow = w.first + row;
  const float c = p.c;

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
  const bool sees = seen > 0;
  const float nl = sees ? -(M + __builtin_amdgcn_logf(L)) / c : -INFINITY, nd = sees ? -delta : 0.f;
  if (hh == 0 && live) { p.nl[stat] = nl; p.nd[stat] = nd; }

  f32x16 acc[MTD];
  clear(acc);
  const bf16_t *kp = p.k + hk * p.k_sh + (int64_t)k_first * p.k_sr, *vp = p.v + hk * p.v_sh + (int64_t)k_first * p.v_sr;
  if (!p.dq) return;
  if (T > 0) {
    const int k_srb = (int)p.k_sr * 2, v_srb = (int)p.v_sr * 2;
    const i32x4 krsrc = packed_rsrc(kp, m, S::ROWB, k_srb), vrsrc = packed_rsrc(vp, m, S::ROWB, v_srb);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(LVAR_LDS char*)smem;
    fill_tile<D, NW>(krsrc, k_srb, 0, lds0, wave, lane);
    fill_tile<D, NW>(vrsrc, v_srb, 0, lds0 + 2 * TILE, wave, lane);
    wait_fills<0>();
    __syncthreads();
    for (int t = 0; t < T; t++) {
      const int par = t & 1;
      // (behind the last tile: rows that nobody reads, or zeros)
      fill_tile<D, NW>(krsrc, k_srb, 64 * (t + 1), lds0 + (1 - par) * TILE, wave, lane);
      fill_tile<D, NW>(vrsrc, v_srb, 64 * (t + 1), lds0 + (3 - par) * TILE, wave, lane);
      const char *kbuf = smem + par * TILE, *vbuf = smem + (2 + par) * TILE;
#pragma unroll
      for (int sub = 0; sub < 2; sub++) {
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 16; i++) { s[i] = nl; dp[i] = nd; }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          s = mfma32(at.rows(kbuf, sub, ks), qf[ks], s);
          dp = mfma32(at.rows(vbuf, sub, ks), gf[ks], dp);
        }
        const int lim = seen - 64 * t - 32 * sub - 4 * hh;
        if (64 * t + 32 * (sub + 1) <= seen_first) {
#pragma unroll
          for (int i = 0; i < 16; i++) s[i] = fast_exp2(s[i] * c) * dp[i];
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float x = fast_exp2(s[i] * c) * dp[i];
            s[i] = 8 * (i >> 2) + (i & 3) < lim ? x : 0.f;
          }
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
          const bf16x8 ds = pack_half(s, kb);
#pragma unroll
          for (int i = 0; i < MTD; i++) acc[i] = mfma32(at.columns(kbuf, 2 * sub + kb, i), ds, acc[i]);
        }
      }
      wait_fills<0>();
      __syncthreads();
    }
  }
  bf16_t* to = p.dq + h * p.dq_sh + (int64_t)(w.first + q0) * p.dq_sr;
  store_rows<D>(smem + wave * (32 * (D * 2 + 16)), acc, p.scale, to, p.dq_sr, w.n - q0, lane);
  if (p.causal) {
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
      a.store(a.a0, p.scale, to + i * p.dq_sr, 0, D);
    }
  }
#endif
}

// ---- dk and dv: 32 keys per wave, tiles of 64 query rows of every query head that shares the key head.  S and dP with the rows of k and v as
// B operands in registers, so a lane owns a key column, and P and dS are in the B operand's layout of dv^T += do^T P and
// dk^T += q^T dS.  The accumulators of S and dP start at -(M + log2 L) / c and -delta of their rows: P is one exp2 of c times the
// sum, dS one product.  SPLIT (head_dim 256): a workgroup accumulates half of the columns of dk and dv, for whole ones take all registers. ----

constexpr int DKV_STAT = 2 * 2 * 64 * 4;   // bytes of the row statistics of two stages

template <int D, int NW, int SPLIT>
__global__ __launch_bounds__(NW * 64, D <= 64 ? 2 : 1) void packed_dkv_kernel(const PackedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = PackedLds<D>;
  constexpr int KS = D / 16, MTD = D / 32 / SPLIT, TILE = S::TILE;
  const int per = p.Hkv * SPLIT;
  const int id = __builtin_amdgcn_workgroup_id_x(), place = id / per, j = id - place * per;
  PackedTile w;
  if (!find_tile<NW * 32>(p.k_off, p.B, p.Tk, place, w)) return;
  const int hk = j / SPLIT, m0 = (j - hk * SPLIT) * MTD;
  const int tid = __builtin_amdgcn_workitem_id_x(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = lane >> 5, r = lane & 31;
  const S at(lane);
  int q_first, n;
  packed_range(p.q_off, w.b, p.T, q_first, n);
  const int k0 = w.row0 + wave * 32, key = min(k0 + r, w.n - 1);
  // rows from `from` on see the lane's key; those of the workgroup's first key come first
  const int shift = w.n - n;
  const int from = p.causal ? max(0, key - shift) : 0;
  const int t0 = p.causal ? min(max(0, w.row0 - shift), n) >> 6 : 0, nT = (n + 63) >> 6, per_head = max(0, nT - t0), steps = per_head * p.G;
  const float c = p.c;

  bf16x8 kf[KS], vf[KS];
  {
    const bf16_t *kp = p.k + hk * p.k_sh + (int64_t)(w.first + key) * p.k_sr + hh * 8, *vp = p.v + hk * p.v_sh + (int64_t)(w.first + key) * p.v_sr + hh * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      kf[ks] = *(const bf16x8*)(kp + ks * 16);
      vf[ks] = *(const bf16x8*)(vp + ks * 16);
    }
  }
  f32x16 dk[MTD], dv[MTD];
  clear(dk);
  clear(dv);
  if (steps > 0) {
    const int q_srb = (int)p.q_sr * 2, g_srb = (int)p.g_sr * 2;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(LVAR_LDS char*)smem;
    float* const stats = (float*)(smem + 4 * TILE);   // [stage parity][-(M + log2 L) / c, -delta][64]
    // stage x: tile t0 + x % per_head of head x / per_head; this thread's statistic of it
    auto stage = [&](int head, int t, int par) -> float {
      const int hq = hk * p.G + head;
      const bf16_t *qp = p.q + hq * p.q_sh + (int64_t)q_first * p.q_sr, *gp = p.g + hq * p.g_sh + (int64_t)q_first * p.g_sr;
      fill_tile<D, NW>(packed_rsrc(qp, n, S::ROWB, q_srb), q_srb, 64 * t, lds0 + par * TILE, wave, lane);
      fill_tile<D, NW>(packed_rsrc(gp, n, S::ROWB, g_srb), g_srb, 64 * t, lds0 + (2 + par) * TILE, wave, lane);
      const int i = 64 * t + (tid & 63);
      const float* from_stat = tid < 64 ? p.nl : p.nd;
      return tid < 128 && i < n ? from_stat[(int64_t)hq * p.T + q_first + i] : tid < 64 ? -INFINITY : 0.f;
    };
    float st = stage(0, t0, 0);
    if (tid < 128) stats[tid] = st;
    wait_fills<0>();
    __syncthreads();
    int head = 0, t = t0;
    for (int x = 0; x < steps; x++) {
      const int par = x & 1;
      int head_n = head, t_n = t + 1;
      if (t_n == nT) { t_n = t0; head_n++; }
      const bool more = x + 1 < steps;
      if (more) st = stage(head_n, t_n, 1 - par);
      const char *qbuf = smem + par * TILE, *gbuf = smem + (2 + par) * TILE;
      const float* sp = stats + par * 128;
#pragma unroll
      for (int sub = 0; sub < 2; sub++) {
        const int i0 = 64 * t + 32 * sub;
        // no row of these sees a key of the wave (its first key is the first to be seen)
        if (i0 >= n || (p.causal && i0 + 31 < k0 - shift)) continue;
        f32x16 s, dp;
#pragma unroll
        for (int a = 0; a < 4; a++) {
          const f32x4 x0 = *(const f32x4*)(sp + 32 * sub + 8 * a + 4 * hh), x1 = *(const f32x4*)(sp + 64 + 32 * sub + 8 * a + 4 * hh);
#pragma unroll
          for (int e = 0; e < 4; e++) { s[4 * a + e] = x0[e]; dp[4 * a + e] = x1[e]; }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          s = mfma32(at.rows(qbuf, sub, ks), kf[ks], s);
          dp = mfma32(at.rows(gbuf, sub, ks), vf[ks], dp);
        }
        if (p.causal && i0 < k0 + 31 - shift) {
          const int lim = from - i0 - 4 * hh;
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const bool sees = 8 * (i >> 2) + (i & 3) >= lim;
            s[i] = sees ? fast_exp2(s[i] * c) : 0.f;
            dp[i] = sees ? s[i] * dp[i] : 0.f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) {
            s[i] = fast_exp2(s[i] * c);
            dp[i] = s[i] * dp[i];
          }
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
          const bf16x8 pb = pack_half(s, kb), db = pack_half(dp, kb);
#pragma unroll
          for (int i = 0; i < MTD; i++) {
            dv[i] = mfma32(at.columns(gbuf, 2 * sub + kb, m0 + i), pb, dv[i]);
            dk[i] = mfma32(at.columns(qbuf, 2 * sub + kb, m0 + i), db, dk[i]);
          }
        }
      }
      if (more && tid < 128) stats[(1 - par) * 128 + tid] = st;
      head = head_n; t = t_n;
      wait_fills<0>();
      __syncthreads();
    }
  }
  constexpr int DW = MTD * 32;   // columns of this workgroup
  char* buf = smem + wave * (32 * (DW * 2 + 16));
  bf16_t* dk_to = p.dk + hk * p.dk_sh + (int64_t)(w.first + k0) * p.dk_sr;
  bf16_t* dv_to = p.dv + hk * p.dv_sh + (int64_t)(w.first + k0) * p.dv_sr;
  if (p.dk) store_rows<DW>(buf, dk, p.scale, dk_to + m0 * 32, p.dk_sr, w.n - k0, lane);
  if (p.dv) store_rows<DW>(buf, dv, 1.f, dv_to + m0 * 32, p.dv_sr, w.n - k0, lane);
  if (p.causal) {
    const bool bad = any_not_finite(dk) | any_not_finite(dv);
    uint64_t keys = __builtin_amdgcn_ballot_w64(bad && k0 + r < w.n);
    keys = (keys | keys >> 32) & 0xffffffffu;
    if (keys) wait_fills<0>();   // the rows as stored above are written again
    while (keys) {
      const int i = __builtin_ctzll(keys);
      keys &= keys - 1;
      const int64_t x = w.first + k0 + i;
      CarefulRow<D, true> a;
      a.clear();
      for (int head = 0; head < p.G; head++) {
        const int hq = hk * p.G + head;
        const int64_t stat = (int64_t)hq * p.T + q_first;
        a.add(p.k + hk * p.k_sh + x * p.k_sr, p.v + hk * p.v_sh + x * p.v_sr, p.q + hq * p.q_sh + (int64_t)q_first * p.q_sr, p.q_sr,
              p.g + hq * p.g_sh + (int64_t)q_first * p.g_sr, p.g_sr, min(__shfl(from, i, 64), n), n, p.nl + stat, p.nd + stat, c);
      }
      if (p.dk) a.store(a.a0, p.scale, dk_to + i * p.dk_sr, m0 * 32, m0 * 32 + DW);
      if (p.dv) a.store(a.a1, 1.f, dv_to + i * p.dv_sr, m0 * 32, m0 * 32 + DW);
    }
  }
#endif
}

template <int D>
static int launch_bwd(PackedParams p, hipStream_t s) {
  constexpr int NW = 4, SPLIT = D > 128 ? 2 : 1;
  constexpr int DQ_LDS = bwd_lds<D>(NW, 0), DKV_LDS = bwd_lds<D>(NW, DKV_STAT);
  const int64_t q_slots = packed_slots(p.T, p.B, NW * 32), k_slots = packed_slots(p.Tk, p.B, NW * 32);
  const int64_t q_groups = q_slots * p.H, k_groups = k_slots * p.Hkv * SPLIT;
  if (q_groups * (NW * 64) > 0xffffffffll || k_groups * (NW * 64) > 0xffffffffll) return LVAR_EINVAL;
  auto dq = packed_dq_kernel<D, NW>;
  auto dkv = packed_dkv_kernel<D, NW, SPLIT>;
  static std::atomic<uint64_t> ready_q{0}, ready_k{0};
  if (!ensure_lds_limit((const void*)dq, DQ_LDS, ready_q) || !ensure_lds_limit((const void*)dkv, DKV_LDS, ready_k)) return LVAR_ELAUNCH;
  p.slots = (int)q_slots;
  hipLaunchKernelGGL(dq, dim3((uint32_t)q_groups), dim3(NW * 64), DQ_LDS, s, p);
  if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (!p.dk && !p.dv) return LVAR_OK;
  p.slots = (int)k_slots;
  hipLaunchKernelGGL(dkv, dim3((uint32_t)k_groups), dim3(NW * 64), DKV_LDS, s, p);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

int launch_packed_bwd(PackedParams p, int head_dim, hipStream_t s) {
  if (head_dim == 128) return launch_bwd<128>(p, s);
  if (head_dim == 64) return launch_bwd<64>(p, s);
  if (head_dim == 256) return launch_bwd<256>(p, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
