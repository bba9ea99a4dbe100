// Attention of the newest tokens over a paged key/value cache, split over the cache's length and joined.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(q_i . k_j * scale * log2e - M_i),  j < limit_i
//
// The rows that share a key/value head (its query heads times the new tokens) are the columns of 16-wide MFMA tiles: with
// S^T = K Q^T the four scores a lane holds are those of keys 4g .. 4g+3 for one query (g = lane / 16), which is the layout that
// the second product O^T = V^T P^T wants its P in, so that scores never leave their lane.  Keys go from memory straight into
// the matrix operand (16 lanes x 64 bytes of 16 rows per load); values are loaded as whole rows (16 lanes cover one row), eight
// rows of a lane are regrouped by byte permutes into pairs of keys, and output columns come out as runs of 32 per lane.  No LDS
// and no barrier in the key loop: a wave waits for nothing but its own loads, and the loads of the next 32 keys are in
// flight while it computes.
//
// The work is (sequence, key/value head, row tile) x stages of 128 keys (32 per wave of a workgroup).  It is cut into pieces
// of about equal length by the lengths that only the device knows: every workgroup scans the lengths and finds its piece.
// The pieces of one tile are joined by a second kernel, in order, so results do not depend on timing.
#include "kvcache.h"

namespace lvar {

constexpr int PA_T = 256, PA_WAVES = 4, PA_STAGE = 128;

// D(16x16) += A(16x32) B(32x16): lane l holds row (column) l % 16, k = 8 * (l / 16) .. + 7; D register r: row 4 * (l / 16) + r, column l % 16.
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float cross_max(float x) {
  int i = __builtin_bit_cast(int, x);
  auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  x = __builtin_fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
  i = __builtin_bit_cast(int, x);
  r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
}
__device__ __forceinline__ float cross_sum(float x) {
  int i = __builtin_bit_cast(int, x);
  auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  x = __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
  i = __builtin_bit_cast(int, x);
  r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
  return __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
}

// ---- the plan: which piece of which sequence a workgroup takes ----

struct Piece {
  int b, len, stages;   // sequence, its length, its stages
  int n, piece;         // pieces per tile of this sequence, which one
  int tile, head;       // row tile, key/value head
  int slot;             // place of its partial result (n > 1)
};

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
  return x;
}
__device__ __forceinline__ int wave_scan(int x, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

__device__ __forceinline__ int stages_of(int len) { return len > 0 ? (len + PA_STAGE - 1) / PA_STAGE : 1; }

// New tokens of sequence b; the rows behind them get an empty result.
__device__ __forceinline__ int fresh_of(const PagedAttnParams& p, int b) { return p.counts ? max(0, min(p.counts[b], p.Lq)) : p.Lq; }

// Length of sequence b within what the table can name.
__device__ __forceinline__ int length_of(const PagedAttnParams& p, int b) { return max(0, min(p.lengths[b], p.max_len)); }

// Stages of a piece: the work spread over `target` pieces, but no less than min_share stages each.  (The launch has checked that
// the stages of all tiles together fit 31 bits.)
__device__ __forceinline__ int share_of(const PagedAttnParams& p, int lane) {
  uint32_t total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) total += wave_sum(b0 + lane < p.B ? stages_of(length_of(p, b0 + lane)) : 0);
  total *= (uint32_t)(p.cache.kv_heads * p.rt);
  return max((int)((total - 1) / (uint32_t)p.target) + 1, p.min_share);
}

// Pieces of a tile of `stages` > 0 stages.
__device__ __forceinline__ int pieces_of(int stages, int share) { return (int)((uint32_t)(stages - 1) / (uint32_t)share) + 1; }

// The piece with number `item`; false behind the last one.  All lanes of a wave call it and get the same answer.
__device__ __forceinline__ bool find_piece(const PagedAttnParams& p, int item, int lane, Piece& out) {
  const int share = share_of(p, lane), units = p.cache.kv_heads * p.rt;
  int before = 0, slots = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    int len = 0, st = 0, n = 0;
    if (b < p.B) {
      len = length_of(p, b);
      st = stages_of(len);
      n = pieces_of(st, share);
    }
    const int mine = n * units, cut = n > 1 ? mine : 0;
    const int upto = wave_scan(mine, lane), cuts = wave_scan(cut, lane);
    const uint64_t hit = __ballot(before + upto > item);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      out.b = b0 + l;
      out.len = __shfl(len, l, 64);
      out.stages = __shfl(st, l, 64);
      out.n = __shfl(n, l, 64);
      const int rest = item - before - __shfl(upto - mine, l, 64);
      out.slot = slots + __shfl(cuts - cut, l, 64) + rest;
      out.tile = rest % p.rt;               // row tiles of the same keys next to each other
      const int hp = rest / p.rt;
      out.piece = hp % out.n;
      out.head = hp / out.n;
      return true;
    }
    before += __shfl(upto, 63, 64);
    slots += __shfl(cuts, 63, 64);
  }
  return false;
}

template <int D, int NT, bool F8, int WAVES_PER_SIMD>
__global__ __launch_bounds__(PA_T, WAVES_PER_SIMD) void paged_attn_kernel(const PagedAttnParams p) {
  constexpr int KS = D / 32;                  // steps of the contraction over the head dimension
  constexpr int CH = D < 128 ? 1 : D / 128;   // chunks of 128 (64) output columns
  constexpr int NE = D < 128 ? D / 16 : 8;    // columns of a chunk per lane and value row
  constexpr int CW = 16 * NE;                 // columns of a chunk
  constexpr int LDO = CW + 4;
  __shared__ float so[PA_WAVES][16][LDO];
  __shared__ float sm[PA_WAVES][NT * 16], sl[PA_WAVES][NT * 16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qi = lane & 15, g = lane >> 4;
  // consecutive pieces (tiles over the same keys) to the same XCD: workgroups are dealt to the 8 of them in turn
  const int per = (gridDim.x + 7) >> 3, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  Piece w;
  if ((int)(blockIdx.x >> 3) >= per || !find_piece(p, item, lane, w)) return;

  const int rows = p.G * p.Lq, row0 = w.tile * NT * 16;
  const int fresh = fresh_of(p, w.b);

  // queries as the second operand, and how many keys each may see
  u32x4 qf[NT][KS];
  int limit[NT];
  int most = 0, least = 0x7fffffff;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int r = row0 + t * 16 + qi, rc = min(r, rows - 1), i = rc / p.G, h = w.head * p.G + (rc - i * p.G);
    const bf16_t* q = p.q + w.b * p.q_sb + h * p.q_sh + i * p.q_sr;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const int d = F8 ? (ks >> 1) * 64 + g * 16 + (ks & 1) * 8 : ks * 32 + g * 8;
      qf[t][ks] = *(const u32x4*)(q + d);
    }
    // (columns behind the last row, and padded rows, go along with the last one: what they compute is not written)
    limit[t] = fresh == 0 ? 0 : p.causal ? max(0, w.len - fresh + min(i, fresh - 1) + 1) : w.len;
    most = max(most, limit[t]);
    least = min(least, limit[t]);
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) {
    most = max(most, __shfl_xor(most, d, 64));
    least = min(least, __shfl_xor(least, d, 64));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);

  const int s0 = (int)((int64_t)w.stages * w.piece / w.n), s1 = (int)((int64_t)w.stages * (w.piece + 1) / w.n);
  const int k_end = min(s1 * PA_STAGE, most);

  f32x4 o[NT][CH][NE] = {};
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) { m[t] = -INFINITY; l[t] = 0.f; }

  const uint8_t* kb = p.cache.k + w.head * p.cache.s_head;
  const uint8_t* vb = p.cache.v + w.head * p.cache.s_head;
  const uint8_t* keb = F8 ? p.cache.k_exp + w.head * p.cache.e_head : nullptr;
  const uint8_t* veb = F8 ? p.cache.v_exp + w.head * p.cache.e_head : nullptr;
  const int32_t* table = p.cache.table + w.b * p.cache.table_stride;
  const int mask = (1 << p.cache.shift) - 1;
  const int sr = (int)p.cache.s_row;

  constexpr int KL = F8 ? KS / 2 : KS;          // 16-byte loads per key row and lane
  u32x4 kf[2][KL];
  u32x4 vr[F8 ? 1 : CH][F8 ? 1 : 8];            // bf16: NE elements of 8 value rows
  u32x2 vc[F8 ? CH : 1][F8 ? 8 : 1];            // e4m3
  uint32_t ke[2], ve[2];

  // page of the 16 keys from `key` on, -1: none
  auto page_of = [&](int key) {
    const int at = min(key >> p.cache.shift, p.cache.max_pages - 1);
    const int pg = table[at];
    return key < k_end && pg >= 0 && pg < p.cache.num_pages ? pg : -1;
  };
  auto load_k = [&](int key, const int* pg) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t pp = pg[j] < 0 ? 0 : pg[j];
      const int slot = (key + 16 * j) & mask;
      const uint8_t* base = kb + pp * p.cache.s_page + (int64_t)slot * p.cache.s_row;
      const uint32_t off = qi * sr + g * 16;
#pragma unroll
      for (int x = 0; x < KL; x++) kf[j][x] = *(const u32x4*)(base + off + x * 64);
      if constexpr (F8) ke[j] = (keb + pp * p.cache.e_page + slot)[qi];
    }
  };
  auto load_v = [&](int key, const int* pg) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t pp = pg[j] < 0 ? 0 : pg[j];
      const int slot = (key + 16 * j) & mask;
      const uint8_t* base = vb + pp * p.cache.s_page + (int64_t)slot * p.cache.s_row;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const uint32_t off = (4 * g + x) * sr + qi * (F8 ? NE : 2 * NE);
#pragma unroll
        for (int c = 0; c < CH; c++) {
          if constexpr (F8) {
            if constexpr (NE == 8) vc[c][4 * j + x] = *(const u32x2*)(base + off + c * 128);
            else vc[c][4 * j + x] = u32x2{*(const uint32_t*)(base + off), 0u};
          } else {
            if constexpr (NE == 8) vr[c][4 * j + x] = *(const u32x4*)(base + off + c * 256);
            else { const u32x2 y = *(const u32x2*)(base + off); vr[c][4 * j + x] = u32x4{y[0], y[1], 0u, 0u}; }
          }
        }
      }
      if constexpr (F8) ve[j] = *(const uint32_t*)(veb + pp * p.cache.e_page + slot + 4 * g);
    }
  };

  int key = s0 * PA_STAGE + wave * 32;
  int pg[2] = {-1, -1};
  if (key < k_end) {
    pg[0] = page_of(key); pg[1] = page_of(key + 16);
    load_k(key, pg);
    load_v(key, pg);
  }
  while (key < k_end) {
    const int next = key + PA_STAGE;
    int npg[2] = {-1, -1};
    if (next < k_end) { npg[0] = page_of(next); npg[1] = page_of(next + 16); }
    const bool ragged = key + 32 > least || pg[0] < 0 || pg[1] < 0;

    // scores
    u32x4 ka[2][KS];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if constexpr (F8) {
        const float sc = exp_value(ke[j]);
#pragma unroll
        for (int x = 0; x < KL; x++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            u32x4 u;
#pragma unroll
            for (int e = 0; e < 2; e++) {
              u[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kf[j][x][2 * h + e], sc, false));
              u[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(kf[j][x][2 * h + e], sc, true));
            }
            ka[j][2 * x + h] = u;
          }
      } else {
#pragma unroll
        for (int x = 0; x < KL; x++) ka[j][x] = kf[j][x];
      }
    }
    u32x4 pf[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float s[8];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) a = mfma16(ka[j][ks], qf[t][ks], a);
#pragma unroll
        for (int r = 0; r < 4; r++) s[4 * j + r] = a[r] * p.c;
      }
      if (ragged) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (pg[j] < 0 || key + 16 * j + 4 * g + r >= limit[t]) s[4 * j + r] = -INFINITY;
      }
      float mt = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3])),
                                 __builtin_fmaxf(__builtin_fmaxf(s[4], s[5]), __builtin_fmaxf(s[6], s[7])));
      mt = __builtin_fmaxf(cross_max(mt), m[t]);
      if (__any(mt > m[t])) {
        const float f = mt == -INFINITY ? 1.f : fast_exp2(m[t] - mt);
        l[t] *= f;
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
          for (int e = 0; e < NE; e++) o[t][c][e] *= f;
        m[t] = mt;
      }
      const float ms = mt == -INFINITY ? 0.f : mt;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        s[e] = fast_exp2(s[e] - ms);
        l[t] += s[e];
      }
      // p is rounded to bf16 for the matrix instruction (its sum is not): 2^-9 per term, independent signs
      pf[t] = pack8u(s);
    }
    if (next < k_end) load_k(next, npg);

    // values: rows of keys nobody may see hold anything, NaN too, and 0 * NaN is not 0
    if (ragged && (key + 32 > k_end || pg[0] < 0 || pg[1] < 0)) {
#pragma unroll
      for (int x = 0; x < 8; x++) {
        const int j = x >> 2;
        const bool dead = pg[j] < 0 || key + 16 * j + 4 * g + (x & 3) >= k_end;
#pragma unroll
        for (int c = 0; c < CH; c++) {
          if constexpr (F8) { if (dead) vc[c][x] = u32x2{0u, 0u}; }
          else { if (dead) vr[c][x] = u32x4{0u, 0u, 0u, 0u}; }
        }
        if constexpr (F8) { if (dead) ve[j] &= ~(0xffu << (8 * (x & 3))); }   // (a leftover byte of 255 stands for infinity)
      }
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
      u32x4 row[8];
#pragma unroll
      for (int x = 0; x < 8; x++) {
        if constexpr (F8) {
          const float sc = exp_value((ve[x >> 2] >> (8 * (x & 3))) & 0xffu);
#pragma unroll
          for (int e = 0; e < NE / 4; e++) {
            row[x][2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc[c][x][e], sc, false));
            row[x][2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vc[c][x][e], sc, true));
          }
        } else {
          row[x] = vr[c][x];
        }
      }
#pragma unroll
      for (int e = 0; e < NE; e++) {
        u32x4 a;
#pragma unroll
        for (int x = 0; x < 4; x++)
          a[x] = __builtin_amdgcn_perm(row[2 * x + 1][e >> 1], row[2 * x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int t = 0; t < NT; t++) o[t][c][e] = mfma16(a, pf[t], o[t][c][e]);
      }
    }
    if (next < k_end) load_v(next, npg);
    pg[0] = npg[0]; pg[1] = npg[1];
    key = next;
  }

  // the four waves' results become one
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const float ls = cross_sum(l[t]);
    if (lane < 16) { sm[wave][t * 16 + qi] = m[t]; sl[wave][t * 16 + qi] = ls; }
  }
  __syncthreads();
  float* slot = w.n > 1 ? p.ws + (int64_t)w.slot * p.slot_rows * (D + 2) : nullptr;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < PA_WAVES; x++) top = __builtin_fmaxf(top, sm[x][t * 16 + qi]);
    const float f = m[t] == -INFINITY ? 0.f : fast_exp2(m[t] - top);
#pragma unroll
    for (int c = 0; c < CH; c++) {
      if (t + c > 0) __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int e = 0; e < NE; e += 4) {
          const f32x4 y = {o[t][c][e][r] * f, o[t][c][e + 1][r] * f, o[t][c][e + 2][r] * f, o[t][c][e + 3][r] * f};
          *(f32x4*)&so[wave][qi][(4 * g + r) * NE + e] = y;
        }
      __syncthreads();
      // thread: query tid / 16, columns NE * (tid % 16) ..
      const int query = threadIdx.x >> 4, col = (threadIdx.x & 15) * NE, r = row0 + t * 16 + query;
      float y[NE] = {};
#pragma unroll
      for (int x = 0; x < PA_WAVES; x++)
#pragma unroll
        for (int e = 0; e < NE; e++) y[e] += so[x][query][col + e];
      float qm = -INFINITY, ql = 0.f;
#pragma unroll
      for (int x = 0; x < PA_WAVES; x++) qm = __builtin_fmaxf(qm, sm[x][t * 16 + query]);
#pragma unroll
      for (int x = 0; x < PA_WAVES; x++) {
        // (no finite score: the sum is 0, or NaN where a score was)
        const float mx = sm[x][t * 16 + query];
        ql += sl[x][t * 16 + query] * (mx == -INFINITY ? 1.f : fast_exp2(mx - qm));
      }
      if (r < rows) {
        if (slot) {
          float* at = slot + (t * 16 + query) * (D + 2);
          if (c == 0 && (threadIdx.x & 15) == 0) { at[D] = qm; at[D + 1] = ql; }
#pragma unroll
          for (int e = 0; e < NE; e += 2) *(f32x2*)(at + c * CW + col + e) = f32x2{y[e], y[e + 1]};
        } else {
          const int i = r / p.G;
          const int64_t out = ((int64_t)w.b * p.H + w.head * p.G + (r - i * p.G)) * p.Lq + i;
          const bool none = i >= fresh || (qm == -INFINITY && ql == 0.f);
          const float inv = 1.f / ql;
#pragma unroll
          for (int e = 0; e < NE; e += 4) {
            const u32x2 u = {pack_bf16(y[e] * inv, y[e + 1] * inv), pack_bf16(y[e + 2] * inv, y[e + 3] * inv)};
            *(u32x2*)(p.o + out * D + c * CW + col + e) = none ? u32x2{0u, 0u} : u;
          }
          if (c == 0 && (threadIdx.x & 15) == 0) { p.M[out] = none ? -INFINITY : qm; p.L[out] = none ? 1.f : ql; }
        }
      }
    }
  }
}

// Joins the pieces of the tiles that were cut: a workgroup per (sequence, key/value head, row), 8 groups of lanes along the pieces.
template <int D>
__global__ __launch_bounds__(512) void paged_join_kernel(const PagedAttnParams p, int tile_rows) {
  constexpr int LPR = D / 4, GR = 512 / LPR;
  __shared__ float so[GR][D];
  __shared__ float sm[GR], sl[GR];
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int tile = row / tile_rows, units = p.cache.kv_heads * p.rt;
  // slots ahead of this sequence
  const int share = share_of(p, lane);
  int n = 0, slots = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int x = b0 + lane;
    const int k = x < p.B ? pieces_of(stages_of(length_of(p, x)), share) : 0;
    slots += wave_sum(x < b && k > 1 ? k * units : 0);
    if (b < b0 + 64) n = __shfl(k, b - b0, 64);
  }
  if (n <= 1) return;
  const float* first = p.ws + ((int64_t)slots + (int64_t)head * n * p.rt + tile) * p.slot_rows * (D + 2) + (row - tile * tile_rows) * (D + 2);
  const int64_t step = (int64_t)p.rt * p.slot_rows * (D + 2);
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
  float top = -INFINITY;
  for (int x = g; x < n; x += GR) top = __builtin_fmaxf(top, first[x * step + D]);
  if (l == 0) sm[g] = top;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < GR; x++) top = __builtin_fmaxf(top, sm[x]);
  float y[4] = {}, sum = 0.f;
#pragma unroll 4
  for (int x = g; x < n; x += GR) {
    const float* at = first + x * step;
    const float mx = at[D], lx = at[D + 1];
    const f32x2 a = *(const f32x2*)(at + l * 4), c = *(const f32x2*)(at + l * 4 + 2);
    const float f = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
    y[0] += a[0] * f; y[1] += a[1] * f; y[2] += c[0] * f; y[3] += c[1] * f;
    sum += mx == -INFINITY ? lx : lx * f;
  }
  if (l == 0) sl[g] = sum;
#pragma unroll
  for (int e = 0; e < 4; e++) so[g][l * 4 + e] = y[e];
  __syncthreads();
  const int i = row / p.G;
  const int64_t out = ((int64_t)b * p.H + head * p.G + (row - i * p.G)) * p.Lq + i;
  float all = 0.f;
#pragma unroll
  for (int x = 0; x < GR; x++) all += sl[x];
  const bool none = i >= fresh_of(p, b) || (top == -INFINITY && all == 0.f);
  for (int col = threadIdx.x; col < D; col += 512) {
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < GR; x++) s += so[x][col];
    p.o[out * D + col] = (bf16_t)(none ? 0.f : s / all);
  }
  if (threadIdx.x == 0) { p.M[out] = none ? -INFINITY : top; p.L[out] = none ? 1.f : all; }
}

// ---- launch ----

struct Shape { int nt, rt, rows, target, min_share; };

static Shape shape_of(int H, int Hkv, int Lq, int head_dim) {
  Shape s;
  const int64_t rows = (int64_t)(H / Hkv) * Lq;
  const int widest = head_dim == 256 ? 2 : 4;
  s.nt = rows <= 16 ? 1 : rows <= 32 ? 2 : widest;
  s.rt = (int)((rows + 16 * s.nt - 1) / (16 * s.nt));
  s.rows = (int)(rows < 16 * s.nt ? rows : 16 * s.nt);
  const int resident = s.nt == 1 ? 3 : s.nt == 2 ? 2 : 1;   // workgroups per compute unit that the registers allow
  s.target = device_cus() * resident;
  s.min_share = 2;
  return s;
}

// Partial results are kept for tiles that are cut only; such a tile has n < 2 * stages / share pieces, so that there are fewer
// than 2 * target of them in all.
int64_t paged_attn_ws_bytes(int B, int H, int Hkv, int Lq, int max_len, int head_dim) {
  const Shape s = shape_of(H, Hkv, Lq, head_dim);
  if (s.target <= 0) return LVAR_ELAUNCH;
  if ((max_len + PA_STAGE - 1) / PA_STAGE <= s.min_share) return 0;   // nothing can be cut
  return 2ll * s.target * s.rows * (head_dim + 2) * 4;
}

template <int D, int NT, bool F8, int W>
static void launch_one(const PagedAttnParams& p, int grid, hipStream_t s) {
  hipLaunchKernelGGL((paged_attn_kernel<D, NT, F8, W>), dim3(grid), dim3(PA_T), 0, s, p);
}

template <int D>
static int launch_d(const PagedAttnParams& p, int nt, hipStream_t s) {
  const bool f8 = p.cache.k_exp != nullptr;
  const int64_t items = (int64_t)p.B * p.cache.kv_heads * p.rt + (p.ws ? p.target : 0);
  if (items > 0x7ffffff0) return LVAR_EINVAL;
  const int grid = (int)((items + 7) / 8 * 8);
  if (nt == 1) f8 ? launch_one<D, 1, true, D == 256 ? 2 : 3>(p, grid, s) : launch_one<D, 1, false, D == 256 ? 2 : 3>(p, grid, s);
  else if (nt == 2) f8 ? launch_one<D, 2, true, D == 256 ? 1 : 2>(p, grid, s) : launch_one<D, 2, false, D == 256 ? 1 : 2>(p, grid, s);
  else if constexpr (D < 256) f8 ? launch_one<D, 4, true, 1>(p, grid, s) : launch_one<D, 4, false, 1>(p, grid, s);
  if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (p.ws) {
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3(p.G * p.Lq, p.cache.kv_heads, p.B), dim3(512), 0, s, p, 16 * nt);
    if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  }
  return LVAR_OK;
}

int launch_paged_attn(PagedAttnParams p, int head_dim, hipStream_t s) {
  const Shape h = shape_of(p.H, p.cache.kv_heads, p.Lq, head_dim);
  if (h.target <= 0) return LVAR_ELAUNCH;
  p.rt = h.rt;
  p.target = h.target;
  p.slot_rows = h.rows;
  // without room for partial results every tile stays whole: a share longer than any sequence
  p.min_share = p.ws ? h.min_share : 0x7fffffff;
  if (head_dim == 128) return launch_d<128>(p, h.nt, s);
  if (head_dim == 64) return launch_d<64>(p, h.nt, s);
  if (head_dim == 256) return launch_d<256>(p, h.nt, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
