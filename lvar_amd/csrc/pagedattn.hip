// Attention of the newest tokens over a paged key/value cache, split over the cache's length and joined.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(q_i . k_j * scale * log2e - M_i),  j < limit_i
//
// The rows that share a key/value head (its query heads times the new tokens) are the columns of 16-wide MFMA tiles: with
// S^T = K Q^T the scores a lane holds are those of keys 4g .. 4g+3 of 16 for one query (g = lane / 16), which is the layout that
// the second product O^T = V^T P^T wants its P in, so that scores never leave their lane.  Two kernels:
//
//   paged_attn_kernel   up to 32 rows, where the cache is read once and its bandwidth is the bound.  Keys go from memory straight into
//     the matrix operand (16 lanes x 64 bytes of 16 rows per load); values are loaded as whole rows (16 lanes cover one row), eight rows
//     of a lane are regrouped by byte permutes into pairs of keys, and output columns come out as runs of 32 per lane.  No
//     LDS and no barrier in the key loop: a wave waits for nothing but its own loads, the loads of its next 32 keys are in flight
//     while it computes, and the four waves take turns at 32 keys.  32 sequences of up to 32768 tokens, 32 query heads over 8 of
//     128: 2.2 GB of bf16 in 395 us (5.6 TB/s; a copy moves 5.2); 131071 tokens in e4m3: 0.27 GB in 55 us.
//   paged_tile_kernel   more rows: keys and values staged in LDS, where the waves share them.  4 x 256 rows of 16 heads over 2521
//     tokens: 45 .. 48 us, 440 .. 470 TFLOP/s.  (With 64 rows per wave and no LDS there is one wave per SIMD and nobody left to
//     compute while it waits: 105 us where this takes 38, 8 sequences of up to 4001 tokens with up to 61 new ones.)
//
// The work is (sequence, key/value head, row tile) x stages of 128 keys.  It is cut into pieces of about equal length by the
// lengths that only the device knows: every workgroup scans the lengths and finds its piece.  The pieces of one tile are joined by
// a second kernel, in order, so results do not depend on timing.
#include "kvcache.h"

namespace lvar {

constexpr int PA_T = 256, PA_WAVES = 4, PA_STAGE = 128;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

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

// bf16 values of 8 codes times a power of two (exact)
__device__ __forceinline__ u32x4 scaled8(u32x2 c, float scale) {
  u32x4 r;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    r[2 * h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], scale, false));
    r[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[h], scale, true));
  }
  return r;
}

// A causal call has keys that some rows of a tile see and others do not.  Their probabilities are 0 for rows that do not, but 0 * inf and
// 0 * NaN are NaN: at the causal border, values that are not finite go into the product as 0, and after the loop they are added one by one to the
// rows that see them (a scan of the border's keys that happens only if there are such values).  The look at the border's values costs 0.2 to 0.5 us of a
// causal call (16 x 8 heads of 32 keys with 8 new tokens 4.84 -> 5.10, 8 x 8 of 64 keys with 40 new tokens 7.87 -> 8.37), staged tiles elsewhere 0.2.
template <class V>
__device__ __forceinline__ void largest(const V& x, u16x2& top) {      // magnitudes of a vector of bf16 pairs, as bits
#pragma unroll
  for (int e = 0; e < (int)(sizeof(V) / 4); e++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu));
}
__device__ __forceinline__ bool odd_pair(u16x2 top) { return top[0] >= 0x7f80 || top[1] >= 0x7f80; }
template <int W, class V>
__device__ __forceinline__ void drop_odd(V& x, uint32_t& any) {        // the infinities and NaN among 2 W bf16 become 0, and `any` not 0
#pragma unroll
  for (int e = 0; e < W; e++) {
    const i16x2 room = i16x2{0x7f7f, 0x7f7f} - __builtin_bit_cast(i16x2, x[e] & 0x7fff7fffu);
    const uint32_t odd = __builtin_bit_cast(uint32_t, room >> 15);     // 0xffff per half
    x[e] &= ~odd;
    any |= odd;
  }
}
// a NaN among 8 codes, or a power of two that takes their largest beyond bf16
__device__ __forceinline__ bool odd_codes(u32x2 c, uint32_t byte) {
  return ((((c[0] & 0x7f7f7f7fu) + 0x01010101u) | ((c[1] & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0 || byte > 246u;
}
// columns col .. col + 3 of a value row where they are not finite, 0 elsewhere
template <bool F8>
__device__ __forceinline__ f32x4 odd_part(const uint8_t* row, float scale, int col) {
  u32x2 x;
  if constexpr (F8) {
    const u32x4 y = scaled8(u32x2{*(const uint32_t*)(row + col), 0u}, scale);
    x = u32x2{y[0], y[1]};
  } else {
    x = *(const u32x2*)(row + 2 * col);
  }
  f32x4 r;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const uint32_t bits = e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16;
    r[e] = __builtin_bit_cast(float, (bits & 0x7f800000u) == 0x7f800000u ? bits : 0u);
  }
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_fmaxf(__builtin_fmaxf(a, b), c); }

// ---- the plan: which piece of which sequence a workgroup takes ----

struct Piece {
  int b, len, stages;   // sequence, its length, its stages
  int n, piece;         // pieces per tile of this sequence, which one
  int tile, head;       // row tile, key/value head
  int rt;               // row tiles with new tokens among their rows
  int slot;             // place of its partial result (n > 1)
  int first_slot;       // of those of its sequence
};

// inclusive prefix sum over a wave
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_mov<0x111>(x);                                                   // row_shr 1, 2, 4, 8: inside rows of 16
  x += dpp_mov<0x112>(x);
  x += dpp_mov<0x114>(x);
  x += dpp_mov<0x118>(x);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);           // row_bcast 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);           // row_bcast 31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

__device__ __forceinline__ int stages_of(int len) { return len > 0 ? (len + PA_STAGE - 1) / PA_STAGE : 1; }

__device__ __forceinline__ const __attribute__((address_space(4))) int32_t* as_constant(const int32_t* p) {
  return (const __attribute__((address_space(4))) int32_t*)(p);
}

// New tokens of a sequence by its entry of `counts`; the rows behind them get an empty result.
__device__ __forceinline__ int fresh_by(const PagedAttnParams& p, int count) { return max(0, min(count, p.Lq)); }
// The same of sequence b, the same one for all lanes: a scalar load.
__device__ __forceinline__ int fresh_of(const PagedAttnParams& p, int b) { return p.counts ? fresh_by(p, as_constant(p.counts)[b]) : p.Lq; }

// Row tiles that hold new tokens (at least one; the rows behind them are written by the last one).
__device__ __forceinline__ int tiles_by(const PagedAttnParams& p, int fresh) { return max(1, (fresh * p.G + p.tile_rows - 1) / p.tile_rows); }
__device__ __forceinline__ int tiles_of(const PagedAttnParams& p, int b) { return p.rt == 1 || !p.counts ? p.rt : tiles_by(p, fresh_by(p, p.counts[b])); }

// Length of sequence b within what the table can name.
__device__ __forceinline__ int length_of(const PagedAttnParams& p, int b) { return max(0, min(p.lengths[b], p.max_len)); }

// Stages of a piece: `total` stages spread over `target` pieces, at least two each if there are more than `singles`.  (The launch has
// checked that the stages of all tiles together fit 31 bits.)
__device__ __forceinline__ int share_of(const PagedAttnParams& p, uint32_t total, uint32_t target) {
  return max((int)((total - 1) / target) + 1, total > p.singles ? 2 : 1);
}

// Pieces of a tile of `stages` > 0 stages if tiles are cut at all; those of up to two stages stay in one.
__device__ __forceinline__ int pieces_of(int stages, int share) {
  return stages <= 2 ? 1 : (int)((uint32_t)(stages - 1) / (uint32_t)share) + 1;
}

// The piece of workgroup `wg`; false for the workgroups that are left over.  All lanes of a wave call it and get the same answer, in
// scalar registers.  Workgroups are dealt to the 8 XCDs in turn; each XCD takes a run of pieces, row tiles over the same keys next to
// each other in one L2.
__device__ __forceinline__ bool find_piece(const PagedAttnParams& p, int wg, int lane, Piece& out) {
  auto take = [&](int pieces, int& item) {
    const int per = (pieces + 7) >> 3;
    item = (wg & 7) * per + (wg >> 3);
    return (wg >> 3) < per && item < pieces;
  };
  auto split = [&](int rest) {              // of the pieces of a sequence
    out.tile = rest % out.rt;
    const int hp = rest / out.rt;
    out.piece = hp % out.n;
    out.head = hp / out.n;
  };
  int item;
  if (!p.ws && (p.rt == 1 || !p.counts)) {
    // nothing is cut and all sequences have the same tiles: no need to look at the others (0.6 us of the 5 us of the smallest calls)
    const int units = p.cache.kv_heads * p.rt;
    if (!take(p.B * units, item)) return false;
    out.b = item / units;
    out.len = max(0, min(as_constant(p.lengths)[out.b], p.max_len));
    out.stages = stages_of(out.len);
    out.n = 1;
    out.rt = p.rt;
    out.slot = out.first_slot = 0;
    split(item - out.b * units);
    return true;
  }
  // (the first 64 sequences are loaded once)
  const int len0 = lane < p.B ? length_of(p, lane) : 0, tiles0 = lane < p.B ? tiles_of(p, lane) : 0;
  int len, st, tiles, n, pieces, share = 0x7fffffff;
  auto look = [&](int b0) {
    const int b = b0 + lane;
    len = b0 == 0 ? len0 : 0;
    tiles = b0 == 0 ? tiles0 : 0;
    if (b0 > 0 && b < p.B) {
      len = length_of(p, b);
      tiles = tiles_of(p, b);
    }
    st = b < p.B ? stages_of(len) : 0;
    n = b < p.B ? pieces_of(st, share) : 0;
  };
  uint32_t total = 0;
  bool cut = false;     // nothing is, or everything may be: with the longest tile the call waits for the join
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    look(b0);
    total += last_lane(wave_scan(st * tiles));
    cut = cut || __any(st > p.whole);
  }
  total *= (uint32_t)p.cache.kv_heads;
  auto count = [&]() {
    pieces = 0;
    for (int b0 = (p.B - 1) & ~63; b0 >= 0; b0 -= 64) {      // (ends with the first 64 in len, st, tiles, n)
      look(b0);
      pieces += last_lane(wave_scan(n * tiles));
    }
    pieces *= p.cache.kv_heads;
  };
  // One round of workgroups, with pieces up to 3 / 8 longer if that makes it one; otherwise fine pieces, whose last round is short.  Lengths
  // that are alike give `target` equal pieces.  Of others some pieces are much longer than the rest, which a round of more workgroups per
  // compute unit evens out if there is enough to do (16 x 8 tiles of up to 2500 keys in bf16, 23.6 -> 21.5 us; of up to 1300 keys with 64
  // rows 22.6 -> 23.4), unless they are so long (32 stages) that their number hardly matters.
  if (cut) share = share_of(p, total, p.target);
  count();
  if (cut && pieces > p.target) {
    const int round = total <= p.some || total > p.most ? p.target : total <= p.many ? p.wide : p.wider;
    const int even = share_of(p, total, round);
    int x = round == p.target ? 1 : 0;
    do {
      share = even + x * max(1, even >> 3);
      count();
    } while (pieces > round && ++x < 4);
    if (pieces > round) {
      share = share_of(p, total, p.finer);
      count();
    }
  }
  if (!take(pieces, item)) return false;
  int before = 0, slots = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (b0 > 0) look(b0);
    const int mine = n * tiles * p.cache.kv_heads, slot = n > 1 ? mine : 0;
    const int upto = wave_scan(mine), cuts = wave_scan(slot);
    const uint64_t hit = __ballot(before + upto > item);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      out.b = b0 + l;
      out.len = __builtin_amdgcn_readlane(len, l);
      out.stages = __builtin_amdgcn_readlane(st, l);
      out.n = __builtin_amdgcn_readlane(n, l);
      out.rt = __builtin_amdgcn_readlane(tiles, l);
      const int rest = item - before - __builtin_amdgcn_readlane(upto - mine, l);
      out.first_slot = slots + __builtin_amdgcn_readlane(cuts - slot, l);
      out.slot = out.first_slot + rest;
      split(rest);
      return true;
    }
    before += last_lane(upto);
    slots += last_lane(cuts);
  }
  return false;
}

// The rows of a padded batch behind the last tile with new tokens: empty results, from the first piece of that tile.
template <int D>
__device__ __forceinline__ void write_padding(const PagedAttnParams& p, const Piece& w) {
  if (w.rt == p.rt || w.piece > 0 || w.tile != w.rt - 1) return;
  const int rows = p.G * p.Lq;
  const int col = threadIdx.x % (D / 8) * 8;
  for (int r = w.rt * p.tile_rows + threadIdx.x / (D / 8); r < rows; r += PA_T / (D / 8)) {   // (rows: their 16-byte pieces may be more than 31 bits)
    const int i = r / p.G;
    const int64_t out = ((int64_t)w.b * p.H + w.head * p.G + (r - i * p.G)) * p.Lq + i;
    *(u32x4*)(p.o + out * D + col) = u32x4{0u, 0u, 0u, 0u};
    if (col == 0) { p.M[out] = -INFINITY; p.L[out] = 1.f; }
  }
}

// What the join needs to know of a sequence, from one of its workgroups.
__device__ __forceinline__ void write_plan(const PagedAttnParams& p, const Piece& w) {
  if (!p.ws || w.piece + w.tile + w.head != 0 || threadIdx.x != 0) return;
  ((int*)p.ws)[2 * w.b] = w.n;
  ((int*)p.ws)[2 * w.b + 1] = w.first_slot;
}

// The end of both kernels.  `so` holds, per wave, 16 rows (16-row group t of the wave's NT) of COLS output columns from col0 on, on
// the scale of the row's maximum over the key waves; sm and sl every wave's maxima and sums.  Adds up the key waves and writes the
// result, or the partial result of a piece.
template <int D, int NT, int RW, int COLS>
__device__ __forceinline__ void write_rows(const PagedAttnParams& p, const Piece& w, int fresh, int t, int col0, const float* so, int ldo,
                                           const float (*sm)[NT * 16], const float (*sl)[NT * 16]) {
  constexpr int KW = PA_WAVES / RW, NC = COLS / 16;
  const int rows = p.G * p.Lq, tile0 = w.tile * NT * RW * 16;
  float* part = w.n > 1 ? p.ws + p.ws_head + (int64_t)w.slot * p.slot_rows * (D + 2) : nullptr;
  // thread: query tid / 16 of every row wave, NC columns
  const int query = threadIdx.x >> 4, col = (threadIdx.x & 15) * NC;
#pragma unroll
  for (int rx = 0; rx < RW; rx++) {
    const int at = rx * NT * 16 + t * 16 + query, r = tile0 + at;   // row of the tile, of the head
    if (r >= rows) break;
    float y[NC] = {}, qm = -INFINITY, ql = 0.f;
#pragma unroll
    for (int x = 0; x < KW; x++) qm = __builtin_fmaxf(qm, sm[x * RW + rx][t * 16 + query]);
#pragma unroll
    for (int x = 0; x < KW; x++) {
#pragma unroll
      for (int e = 0; e < NC; e++) y[e] += so[((x * RW + rx) * 16 + query) * ldo + col + e];
      const float mx = sm[x * RW + rx][t * 16 + query];
      ql += sl[x * RW + rx][t * 16 + query] * (mx == -INFINITY ? 1.f : fast_exp2(mx - qm));
    }
    if (part) {
      float* to = part + at * (D + 2);
      if (col0 == 0 && col == 0) { to[D] = qm; to[D + 1] = ql; }
#pragma unroll
      for (int e = 0; e < NC; e += 2) *(f32x2*)(to + col0 + col + e) = f32x2{y[e], y[e + 1]};
    } else {
      const int i = r / p.G;
      const int64_t out = ((int64_t)w.b * p.H + w.head * p.G + (r - i * p.G)) * p.Lq + i;
      const bool none = i >= fresh || (qm == -INFINITY && ql == 0.f);
      const float inv = 1.f / ql;
#pragma unroll
      for (int e = 0; e < NC; e += 4) {
        const u32x2 u = {pack_bf16(y[e] * inv, y[e + 1] * inv), pack_bf16(y[e + 2] * inv, y[e + 3] * inv)};
        *(u32x2*)(p.o + out * D + col0 + col + e) = none ? u32x2{0u, 0u} : u;
      }
      if (col0 == 0 && col == 0) { p.M[out] = none ? -INFINITY : qm; p.L[out] = none ? 1.f : ql; }
    }
  }
}

// Keys that row r of a head sees, and whether that is fewer for earlier rows.  (Rows behind the last one, and padded rows, go along
// with the last one: what they compute is not written.)
__device__ __forceinline__ int limit_of(const PagedAttnParams& p, const Piece& w, int fresh, int r) {
  const int i = min(r, p.G * p.Lq - 1) / p.G;
  return fresh == 0 ? 0 : p.causal ? max(0, w.len - fresh + min(i, fresh - 1) + 1) : w.len;
}

// One step of the running softmax of 16 rows over the NS scores of a lane: afterwards s holds the exponentials.  m: what they count
// from, the same for the four lanes of a query; l: their sum in this lane; top: its largest score.  The reference moves when
// a score is more than 2^8 above it (or is the first): sums and outputs stay far from the ends of 32-bit range, and the exchange
// between lanes and the rescaling of the outputs are rare.
template <int NS, int NO>
__device__ __forceinline__ void softmax_step(float* s, float c, float& m, float& l, float& top, f32x4* o) {
  float mt = __builtin_fmaxf(s[0], s[1]);
#pragma unroll
  for (int e = 2; e < NS; e += 2) mt = max3(mt, s[e], s[e + 1]);
  top = __builtin_fmaxf(top, mt);
  if (__any(mt * c > m + 8.f)) {
    mt = __builtin_fmaxf(cross_max(mt) * c, m);
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - mt);
    l *= f;
#pragma unroll
    for (int e = 0; e < NO; e++) o[e] *= f;
    m = mt;
  }
  const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int e = 0; e < NS; e++) {
    s[e] = fast_exp2(__builtin_fmaf(s[e], c, -ms));
    l += s[e];
  }
}

// Puts a wave's sums on the scale of its true maximum (the M of the result): writes both, and returns the factor for its outputs
// in m and the maximum in top.
__device__ __forceinline__ void settle(float c, int lane, float& m, float& l, float& top, float* sm, float* sl) {
  const float mx = cross_max(top) * c, ls = cross_sum(l);
  // (no finite score: nothing, or NaN that has to stay one)
  const float f = m == -INFINITY ? 1.f : fast_exp2(m - mx);
  if (lane < 16) { sm[lane] = mx; sl[lane] = ls * f; }
  m = f;
  top = mx;
}

template <int D, int NT, bool F8, int WAVES_PER_SIMD>
__global__ __launch_bounds__(PA_T, WAVES_PER_SIMD) void paged_attn_kernel(const PagedAttnParams p) {
  constexpr int KS = D / 32;                  // steps of the contraction over the head dimension
  constexpr int CH = D < 128 ? 1 : D / 128;   // chunks of 128 (64) output columns
  constexpr int NE = D < 128 ? D / 16 : 8;    // columns of a chunk per lane and value row
  constexpr bool TWO = D < 256 || F8;         // the exponentials as two bf16 terms
  constexpr int CW = 16 * NE;                 // columns of a chunk
  constexpr int LDO = CW + 4;
  __shared__ float so[PA_WAVES][16][LDO];
  __shared__ float sm[PA_WAVES][NT * 16], sl[PA_WAVES][NT * 16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qi = lane & 15, g = lane >> 4;
  Piece w;
  if (!find_piece(p, blockIdx.x, lane, w)) return;
  write_plan(p, w);

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
    limit[t] = limit_of(p, w, fresh, r);
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
  float m[NT], l[NT], top[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) { m[t] = top[t] = -INFINITY; l[t] = 0.f; }

  const uint8_t* kb = p.cache.k + w.head * p.cache.s_head;
  const uint8_t* vb = p.cache.v + w.head * p.cache.s_head;
  const uint8_t* keb = F8 ? p.cache.k_exp + w.head * p.cache.e_head : nullptr;
  const uint8_t* veb = F8 ? p.cache.v_exp + w.head * p.cache.e_head : nullptr;
  // through the constant address space: scalar loads, which do not stand in the queue of the vector loads
  const __attribute__((address_space(4))) int32_t* table = as_constant(p.cache.table + w.b * p.cache.table_stride);
  const int mask = (1 << p.cache.shift) - 1;
  const int sr = (int)p.cache.s_row;

  constexpr int KL = F8 ? KS / 2 : KS;          // 16-byte loads per key row and lane
  u32x4 kf[2][KL];
  using Row = std::conditional_t<NE == 8, u32x4, u32x2>;
  Row vr[F8 ? 1 : CH][F8 ? 1 : 8];              // bf16: NE elements of 8 value rows
  u32x2 vc[F8 ? CH : 1][F8 ? 8 : 1];            // e4m3
  uint32_t ke[2], ve[2];

  // table entry for the 16 keys from `key` on (in the table whatever the key), and the page that it names, -1: none
  auto entry_of = [&](int key) { return table[min(key >> p.cache.shift, p.cache.max_pages - 1)]; };
  auto page_of = [&](int key, int entry) { return key < k_end && entry >= 0 && entry < p.cache.num_pages ? entry : -1; };
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
            vr[c][4 * j + x] = *(const Row*)(base + off + c * 256);
          }
        }
      }
      if constexpr (F8) ve[j] = *(const uint32_t*)(veb + pp * p.cache.e_page + slot + 4 * g);
    }
  };

  constexpr int STEP = 32 * PA_WAVES;
  int key = s0 * PA_STAGE + wave * 32;
  int pg[2] = {-1, -1}, entry[2] = {0, 0};   // entry: of the next 32 keys
  uint64_t odd = 0;                          // lanes that dropped values
  if (key < k_end) {
    pg[0] = page_of(key, entry_of(key)); pg[1] = page_of(key + 16, entry_of(key + 16));
    load_k(key, pg);
    load_v(key, pg);
    entry[0] = entry_of(key + STEP); entry[1] = entry_of(key + STEP + 16);
  }
  while (key < k_end) {
    const int next = key + STEP;
    const int npg[2] = {page_of(next, entry[0]), page_of(next + 16, entry[1])};
    entry[0] = entry_of(next + STEP); entry[1] = entry_of(next + STEP + 16);
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
    u32x4 pf[NT], pl[TWO ? NT : 1];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float s[8];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) a = mfma16(ka[j][ks], qf[t][ks], a);
#pragma unroll
        for (int r = 0; r < 4; r++) s[4 * j + r] = a[r];
      }
      if (ragged) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (pg[j] < 0 || key + 16 * j + 4 * g + r >= limit[t]) s[4 * j + r] = -INFINITY;
      }
      softmax_step<8, CH * NE>(s, p.c, m[t], l[t], top[t], &o[t][0][0]);
      // p goes into the matrix instruction as two bf16 terms, which leave at most 2^-16 of it out: the result is off by its own rounding only (rms 0.0017
      // of it instead of 0.0023; a product more per value, 2 % of short calls).  256 columns of bf16 have no registers for the second: up to 2^-8 there.
      pf[t] = pack8u(s);
      if constexpr (TWO) {
        float back[8];
        unpack8(pf[t], back);
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] -= back[e];
        pl[t] = pack8u(s);
      }
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
          else { if (dead) vr[c][x] = Row{}; }
        }
        if constexpr (F8) { if (dead) ve[j] &= ~(0xffu << (8 * (x & 3))); }   // (a leftover byte of 255 stands for infinity)
      }
    }
    const bool border = least < k_end && key + 32 > least;   // some rows see these keys and others do not
    if constexpr (!F8) {
      if (border) {
        uint32_t some = 0;
#pragma unroll
        for (int x = 0; x < 8; x++)
#pragma unroll
          for (int c = 0; c < CH; c++) {
            drop_odd<NE / 2>(vr[c][x], some);
            if constexpr (D > 64) __builtin_amdgcn_sched_barrier(0);   // (rows side by side take registers that the loop does not have)
          }
        odd |= __ballot(some != 0);
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
#pragma unroll
          for (int e = 0; e < NE / 2; e++) row[x][e] = vr[c][x][e];
        }
      }
      if constexpr (F8) {
        if (border) {
          uint32_t some = 0;
#pragma unroll
          for (int x = 0; x < 8; x++) drop_odd<NE / 2>(row[x], some);
          odd |= __ballot(some != 0);
        }
      }
#pragma unroll
      for (int e = 0; e < NE; e++) {
        u32x4 a;
#pragma unroll
        for (int x = 0; x < 4; x++)
          a[x] = __builtin_amdgcn_perm(row[2 * x + 1][e >> 1], row[2 * x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          o[t][c][e] = mfma16(a, pf[t], o[t][c][e]);
          if constexpr (TWO) o[t][c][e] = mfma16(a, pl[t], o[t][c][e]);
        }
      }
    }
    if (next < k_end) load_v(next, npg);
    pg[0] = npg[0]; pg[1] = npg[1];
    key = next;
  }
  if (__builtin_expect(odd != 0, false)) {
#pragma unroll 1
    for (int at = max(s0 * PA_STAGE, least & ~31); at < k_end; at++) {
      const int page = page_of(at, entry_of(at)), slot = at & mask;
      if (page < 0 || ((at >> 5) & (PA_WAVES - 1)) != wave) continue;
      const uint8_t* from = vb + page * p.cache.s_page + slot * p.cache.s_row;
      const float sc = F8 ? exp_value((veb + page * p.cache.e_page)[slot]) : 0.f;
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int e = 0; e < NE; e += 4) {
            const f32x4 y = odd_part<F8>(from, sc, c * CW + (4 * g + r) * NE + e);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
              for (int i = 0; i < 4; i++) o[t][c][e + i][r] += at < limit[t] ? y[i] : 0.f;
          }
    }
  }

  // the waves' results become one
#pragma unroll
  for (int t = 0; t < NT; t++) settle(p.c, lane, m[t], l[t], top[t], &sm[wave][t * 16], &sl[wave][t * 16]);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; t++) {
    float best = -INFINITY;
#pragma unroll
    for (int x = 0; x < PA_WAVES; x++) best = __builtin_fmaxf(best, sm[x][t * 16 + qi]);
    const float f = top[t] == -INFINITY ? 1.f : m[t] * fast_exp2(top[t] - best);
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
      write_rows<D, NT, 1, CW>(p, w, fresh, t, c * CW, &so[0][0][0], LDO, sm, sl);
    }
  }
}

// ---- many rows per key/value head ----

__device__ __forceinline__ u32x2 read_tr(LVAR_LDS const char* p) {   // see lds_read_tr
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LVAR_LDS bf16x4*)p));
}

// The same with keys and values staged in LDS, where the waves of a workgroup share them: RW row waves of 16 * NT rows, 4 / RW key
// waves of 32 keys of a tile of KT.  A quarter of the tile goes through the registers of each wave (requested a tile ahead,
// converted there if it is e4m3, masked there if nobody may see it), into the buffer that nobody reads: one barrier per tile.
// 16-byte pieces of a row change places by their row number so that 16 keys (first product) and 16 rows of 32 bytes (transposing
// reads of the second) lie in different banks.
template <int D, int NT, int RW, bool F8>
__global__ __launch_bounds__(PA_T, 2) void paged_tile_kernel(const PagedAttnParams p) {
  constexpr int KT = D == 256 ? 32 : 64, KW = PA_WAVES / RW, KS = D / 32, NB = D / 16;
  constexpr int RB = 2 * D, BUF = KT * RB;                  // bytes of a row, of a tile of keys or values
  constexpr int LPW = D / 8, RPI = 64 / LPW, NI = KT / 4 / RPI;   // fills: lanes per row, rows per load, loads per wave
  constexpr int HALVES = KT / (32 * KW);                    // runs of 32 keys per wave and tile
  static_assert(HALVES >= 1, "a wave takes 32 keys");
  constexpr int LDO = D + 4;
  extern __shared__ __align__(16) char smem[];              // [2 buffers][keys, values][BUF]; then the outputs
  __shared__ float sm[PA_WAVES][NT * 16], sl[PA_WAVES][NT * 16];
  __shared__ __align__(4) uint8_t missing[2][4];             // quarters of a tile: 1 without a page (or behind the last key), 2 with values that were dropped

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, kw = wave / RW;
  const int qi = lane & 15, g = lane >> 4;
  Piece w;
  if (!find_piece(p, blockIdx.x, lane, w)) return;
  write_plan(p, w);

  const int rows = p.G * p.Lq, tile0 = w.tile * NT * RW * 16, row0 = tile0 + rw * NT * 16;
  const int fresh = fresh_of(p, w.b);
  const int s0 = (int)((int64_t)w.stages * w.piece / w.n), s1 = (int)((int64_t)w.stages * (w.piece + 1) / w.n);
  // limits do not fall from row to row: the last row of the tile, and of the wave, has the largest
  const int k_end = min(s1 * PA_STAGE, limit_of(p, w, fresh, min(tile0 + NT * RW * 16, rows) - 1));
  const int least = limit_of(p, w, fresh, row0);
  const int lowest = p.causal ? max(0, w.len - fresh) : 0x7fffffff;   // keys that all rows see (new tokens aside)
  const int mine = row0 < fresh * p.G ? limit_of(p, w, fresh, row0 + NT * 16 - 1) : 0;   // a wave without new rows only fills

  u32x4 qf[NT][KS];
  int limit[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int r = row0 + t * 16 + qi, rc = min(r, rows - 1), i = rc / p.G, h = w.head * p.G + (rc - i * p.G);
    const bf16_t* q = p.q + w.b * p.q_sb + h * p.q_sh + i * p.q_sr;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) qf[t][ks] = *(const u32x4*)(q + ks * 32 + g * 8);
    limit[t] = limit_of(p, w, fresh, r);
  }

  f32x4 o[NT][NB] = {};
  float m[NT], l[NT], top[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) { m[t] = top[t] = -INFINITY; l[t] = 0.f; }

  // fills
  const uint8_t* kb = p.cache.k + w.head * p.cache.s_head;
  const uint8_t* vb = p.cache.v + w.head * p.cache.s_head;
  const uint8_t* keb = F8 ? p.cache.k_exp + w.head * p.cache.e_head : nullptr;
  const uint8_t* veb = F8 ? p.cache.v_exp + w.head * p.cache.e_head : nullptr;
  const __attribute__((address_space(4))) int32_t* table = as_constant(p.cache.table + w.b * p.cache.table_stride);
  const int mask = (1 << p.cache.shift) - 1, sr = (int)p.cache.s_row;
  const int fr = lane / LPW, fc = lane % LPW;               // row of a load, 16-byte piece (of bf16) of the row
  auto entry_of = [&](int key) { return table[min(key >> p.cache.shift, p.cache.max_pages - 1)]; };
  auto page_of = [&](int key, int entry) { return key < k_end && entry >= 0 && entry < p.cache.num_pages ? entry : -1; };
  struct Fill {                                             // a wave's quarter of a tile on its way
    u32x4 row[F8 ? 1 : 2][F8 ? 1 : NI];
    u32x2 code[F8 ? 2 : 1][F8 ? NI : 1];
    uint32_t byte[F8 ? 2 : 1][F8 ? NI : 1];
    int page;
  };
  // Quarter of the tile from `key` on; behind the last tile that one again (nobody reads it): no branch stands between the loads
  // of one tile and the next, so that the wait for one never waits for the other.
  const int k0 = s0 * PA_STAGE, last = k_end > k0 ? (k_end - 1) / KT * KT : k0;
  auto quarter_of = [&](int key) { return min(key, last) + wave * (KT / 4); };
  auto request = [&](Fill& f, int key, int entry) {
    const int first = quarter_of(key);
    f.page = page_of(first, entry);
    const int64_t pp = f.page < 0 ? 0 : f.page;
    const int slot = first & mask;
    const int64_t base = pp * p.cache.s_page + (int64_t)slot * p.cache.s_row;
#pragma unroll
    for (int x = 0; x < NI; x++) {
      const uint32_t off = (x * RPI + fr) * sr + fc * (F8 ? 8 : 16);
      if constexpr (F8) {
        f.code[0][x] = *(const u32x2*)(kb + base + off);
        f.code[1][x] = *(const u32x2*)(vb + base + off);
        f.byte[0][x] = (keb + pp * p.cache.e_page + slot)[x * RPI + fr];
        f.byte[1][x] = (veb + pp * p.cache.e_page + slot)[x * RPI + fr];
      } else {
        f.row[0][x] = *(const u32x4*)(kb + base + off);
        f.row[1][x] = *(const u32x4*)(vb + base + off);
      }
    }
  };
  auto deposit = [&](const Fill& f, int key, int buf) {
    const int first = quarter_of(key);
    const bool ragged = first + KT / 4 > k_end || f.page < 0;
    auto value_of = [&](int x) {
      u32x4 vx;
      if constexpr (F8) vx = scaled8(f.code[1][x], exp_value(f.byte[1][x]));
      else vx = f.row[1][x];
      // rows of keys nobody may see hold anything, NaN too, and 0 * NaN is not 0
      if (ragged && (f.page < 0 || first + x * RPI + fr >= k_end)) vx = u32x4{0u, 0u, 0u, 0u};
      return vx;
    };
    auto place_of = [&](int x, bool values) {
      const int row = wave * (KT / 4) + x * RPI + fr;
      const int kc = fc ^ (D == 64 ? (row >> 1) & 7 : row & 15), vc = fc ^ (D == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1);
      return (u32x4*)(smem + (2 * buf + (values ? 1 : 0)) * BUF + row * RB + (values ? vc : kc) * 16);
    };
#pragma unroll
    for (int x = 0; x < NI; x++) {
      if constexpr (F8) *place_of(x, false) = scaled8(f.code[0][x], exp_value(f.byte[0][x]));
      else *place_of(x, false) = f.row[0][x];
      *place_of(x, true) = value_of(x);
    }
    uint32_t flags = f.page < 0 ? 1u : 0u;
    if (__builtin_expect(first + KT / 4 > lowest, false)) {
      bool odd = false;
      u16x2 top = {0, 0};
#pragma unroll
      for (int x = 0; x < NI; x++) {
        if constexpr (F8) odd = odd || odd_codes(f.code[1][x], f.byte[1][x]);
        else largest(f.row[1][x], top);
      }
      if (__builtin_expect(__any(odd || odd_pair(top)), false)) {   // once more, without them
        uint32_t some = 0;
#pragma unroll
        for (int x = 0; x < NI; x++) {
          u32x4 vx = value_of(x);
          drop_odd<4>(vx, some);
          *place_of(x, true) = vx;
        }
        if (__any(some != 0)) flags |= 2u;
      }
    }
    if (lane == 0) missing[buf][wave] = (uint8_t)flags;
  };

  // addresses of the reads: constants of a product's steps are exclusive-ored in, rows added
  const int ka = qi * RB + (g ^ (D == 64 ? (qi >> 1) & 3 : qi & 3)) * 16 + ((D == 64 ? qi >> 3 : qi >> 2) << 6);
  const int vrow = 4 * g + (qi >> 2);
  const int va = vrow * RB + (D == 64 ? (vrow >> 1) & 3 : vrow & 7) * 32 + (qi & 3) * 8;
  LVAR_LDS const char *const lds = (LVAR_LDS const char*)smem, *kp[KS], *vp[NB];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) kp[ks] = lds + (ka ^ (ks * 64)) + kw * HALVES * 32 * RB;
#pragma unroll
  for (int n = 0; n < NB; n++) vp[n] = lds + (va ^ (n * 32)) + kw * HALVES * 32 * RB;

  uint32_t dropped = 0;                                     // values of the causal border
  auto compute = [&](int key, int buf) {
    const uint32_t gone = *(const uint32_t*)missing[buf];
#pragma unroll
    for (int hh = 0; hh < HALVES; hh++) {
      const int run = (kw * HALVES + hh) * 32, first = key + run;
      if (first >= mine) continue;
      u32x4 pf[NT];
      f32x4 a[NT][2] = {};
      // (all reads of a run of steps ahead of its products: a wave has one other to hide their time behind)
      constexpr int KG = KS > 4 ? 4 : KS;
#pragma unroll
      for (int k1 = 0; k1 < KS; k1 += KG) {
        u32x4 kx[KG][2];
#pragma unroll
        for (int ks = 0; ks < KG; ks++)
#pragma unroll
          for (int j = 0; j < 2; j++) kx[ks][j] = *(LVAR_LDS const u32x4*)(kp[k1 + ks] + 2 * buf * BUF + (hh * 32 + 16 * j) * RB);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < KG; ks++)
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int t = 0; t < NT; t++) a[t][j] = mfma16(kx[ks][j], qf[t][k1 + ks], a[t][j]);
      }
      __builtin_amdgcn_s_setprio(0);
      const bool ragged = first + 32 > least || __builtin_amdgcn_readfirstlane(gone) != 0;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = a[t][e >> 2][e & 3];
        if (ragged) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int at = run + 16 * (e >> 2);             // of the tile: the 16 keys of one page
            if (((gone >> (at / (KT / 4) * 8)) & 1) || key + at + 4 * g + (e & 3) >= limit[t]) s[e] = -INFINITY;
          }
        }
        softmax_step<8, NB>(s, p.c, m[t], l[t], top[t], o[t]);
        // (one bf16 term: off by up to 2^-8 each, with independent signs; their sum is not rounded.  A second term is half as many products again, and those
        // are among the bounds here: 8 x 8 ragged tiles of 61 new tokens 51.2 -> 59.8 us, 4 x 16 heads of 2521 keys with 256 rows 46.9 -> 53.9)
        pf[t] = pack8u(s);
      }
      u32x4 vx[2][4];
      auto read4 = [&](int n0, u32x4* to) {
#pragma unroll
        for (int n = 0; n < 4; n++) {
          LVAR_LDS const char* at = vp[n0 + n] + (2 * buf + 1) * BUF + hh * 32 * RB;
          const u32x2 lo = read_tr(at), hi = read_tr(at + 16 * RB);
          to[n] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      };
      read4(0, vx[0]);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int n0 = 0; n0 < NB; n0 += 4) {
        if (n0 + 4 < NB) read4(n0 + 4, vx[(n0 / 4 + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int t = 0; t < NT; t++) o[t][n0 + n] = mfma16(vx[(n0 / 4) & 1][n], pf[t], o[t][n0 + n]);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    dropped |= __builtin_amdgcn_readfirstlane(gone) & 0x02020202u;
  };

  // (the table entry that the next request needs is loaded ahead of a barrier: scalar loads and LDS reads share a counter)
  Fill f;
  request(f, k0, entry_of(quarter_of(k0)));
  deposit(f, k0, 0);
  int entry = entry_of(quarter_of(k0 + KT));
  __syncthreads();
  for (int key = k0; key < k_end; key += 2 * KT) {
    request(f, key + KT, entry);
    compute(key, 0);
    deposit(f, key + KT, 1);
    entry = entry_of(quarter_of(key + 2 * KT));
    __syncthreads();
    request(f, key + 2 * KT, entry);
    if (key + KT < k_end) compute(key + KT, 1);
    deposit(f, key + 2 * KT, 0);
    entry = entry_of(quarter_of(key + 3 * KT));
    __syncthreads();
  }
  if (__builtin_expect(dropped != 0, false)) {
#pragma unroll 1
    for (int at = max(k0, lowest & ~31); at < k_end; at++) {
      const int page = page_of(at, entry_of(at)), slot = at & mask;
      if (page < 0 || at / 32 % (KT / 32) / HALVES != kw) continue;
      const uint8_t* from = vb + page * p.cache.s_page + slot * p.cache.s_row;
      const float sc = F8 ? exp_value((veb + page * p.cache.e_page)[slot]) : 0.f;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        const f32x4 y = odd_part<F8>(from, sc, n * 16 + 4 * g);
#pragma unroll
        for (int t = 0; t < NT; t++) o[t][n] += at < limit[t] ? y : f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }

#pragma unroll
  for (int t = 0; t < NT; t++) settle(p.c, lane, m[t], l[t], top[t], &sm[wave][t * 16], &sl[wave][t * 16]);
  __syncthreads();
  float* so = (float*)smem;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    float best = -INFINITY;
#pragma unroll
    for (int x = 0; x < KW; x++) best = __builtin_fmaxf(best, sm[x * RW + rw][t * 16 + qi]);
    const float f = top[t] == -INFINITY ? 1.f : m[t] * fast_exp2(top[t] - best);
    if (t > 0) __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; n++) *(f32x4*)&so[(wave * 16 + qi) * LDO + n * 16 + 4 * g] = o[t][n] * f;
    __syncthreads();
    write_rows<D, NT, RW, D>(p, w, fresh, t, 0, so, LDO, sm, sl);
  }
  write_padding<D>(p, w);
}

// Joins the pieces of the tiles that were cut, in order.  A workgroup takes 512 / (D / 4) groups of D / 4 lanes: RPB rows with
// GR / RPB groups each along the pieces.
template <int D, int RPB>
__global__ __launch_bounds__(512) void paged_join_kernel(const PagedAttnParams p) {
  constexpr int LPR = D / 4, GR = 512 / LPR, GP = GR / RPB;
  static_assert(GR % RPB == 0, "groups per row");
  __shared__ float so[GP > 1 ? GR : 1][D];
  __shared__ float sm[GR], sl[GR];
  const int head = blockIdx.y, b = blockIdx.z;
  const int n = ((const int*)p.ws)[2 * b];
  if (n <= 1) return;
  const int first_slot = ((const int*)p.ws)[2 * b + 1];
  const int l = threadIdx.x % LPR, g = threadIdx.x / LPR, x0 = g / RPB;
  const int fresh = fresh_of(p, b), rt = tiles_by(p, fresh), rows = min(p.G * p.Lq, rt * p.tile_rows);   // (the rows behind these are written)
  if ((int)blockIdx.x * RPB >= rows) return;
  const int row = blockIdx.x * RPB + g % RPB, rc = min(row, rows - 1), tile = rc / p.tile_rows;
  const float* first = p.ws + p.ws_head + ((int64_t)(first_slot + head * n * rt + tile) * p.slot_rows + (rc - tile * p.tile_rows)) * (D + 2);
  const int64_t step = (int64_t)rt * p.slot_rows * (D + 2);
  // a running maximum, sum and output per group, four pieces in flight
  float top = -INFINITY, sum = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int x = x0; x < n; x += 4 * GP) {
    float mx[4], lx[4];
    f32x2 lo[4], hi[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const float* at = first + min(x + u * GP, n - 1) * step;
      mx[u] = at[D]; lx[u] = at[D + 1];
      lo[u] = *(const f32x2*)(at + l * 4); hi[u] = *(const f32x2*)(at + l * 4 + 2);
    }
    float best = top;
#pragma unroll
    for (int u = 0; u < 4; u++) best = __builtin_fmaxf(best, mx[u]);   // (a piece that is looked at twice does not change it)
    const float fade = top == -INFINITY ? 1.f : fast_exp2(top - best);
    y *= fade; sum *= fade; top = best;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if (x + u * GP >= n) break;
      const float f = mx[u] == -INFINITY ? 1.f : fast_exp2(mx[u] - top);   // (no finite score: zeros, or NaN that stays one)
      y += f32x4{lo[u][0], lo[u][1], hi[u][0], hi[u][1]} * f;
      sum += lx[u] * f;
    }
  }
  if constexpr (GP > 1) {
    if (l == 0) { sm[g] = top; sl[g] = sum; }
    *(f32x4*)&so[g][l * 4] = y;
    __syncthreads();
    if (g >= RPB) return;
#pragma unroll
    for (int x = 0; x < GP; x++) top = __builtin_fmaxf(top, sm[x * RPB + g]);
    sum = 0.f;
    y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < GP; x++) {
      const float mx = sm[x * RPB + g], f = mx == -INFINITY ? 1.f : fast_exp2(mx - top);
      sum += sl[x * RPB + g] * f;
      y += *(const f32x4*)&so[x * RPB + g][l * 4] * f;
    }
  }
  if (row >= rows) return;
  const int i = row / p.G;
  const int64_t out = ((int64_t)b * p.H + head * p.G + (row - i * p.G)) * p.Lq + i;
  const bool none = i >= fresh || (top == -INFINITY && sum == 0.f);
  const float inv = 1.f / sum;
  const u32x2 u = {pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv)};
  *(u32x2*)(p.o + out * D + l * 4) = none ? u32x2{0u, 0u} : u;
  if (l == 0) { p.M[out] = none ? -INFINITY : top; p.L[out] = none ? 1.f : sum; }
}

// ---- launch ----

struct Shape { int cus, nt, rw, rt, rows, whole, finer; bool staged; };

// Rows per tile: 16 up to 16 rows of a key/value head, 32 up to 32 (each wave reads keys for itself), more with staged tiles: 64 up to
// 64 rows, then 128 (head_dim 256: 64 from 17 rows on, its outputs take twice the registers).
static Shape shape_of(int B, int H, int Hkv, int Lq, int head_dim) {
  Shape s;
  s.cus = device_cus();
  const int64_t rows = (int64_t)(H / Hkv) * Lq;
  s.nt = rows <= 16 || head_dim == 256 ? 1 : 2;
  s.staged = rows > 16 * s.nt;
  s.rw = !s.staged ? 1 : rows <= 64 && head_dim < 256 ? 2 : 4;
  const int tile = 16 * s.nt * s.rw;
  s.rt = (int)((rows + tile - 1) / tile);
  s.rows = (int)(rows < tile ? rows : tile);
  // Calls whose tiles all have up to this many stages are not cut.  Cutting costs the join and the partial results, 4 to 6 us with few tiles and more with many;
  // it saves the stages that a workgroup does not do: 0.65, 1.1 and 2.5 us each (head_dim 64, 128, 256), 1.5, 2.1 and 3.8 of staged
  // tiles.  The limits are where both measured the same (uncut / cut at 4 stages, 16 heads of 64 rows: head_dim 64 11.7 / 12.1, 128 15.4 / 14.0,
  // 256 22.2 / 17.8; of 1 row: head_dim 256 16.0 / 11.5), as measured with 1 / 16 to all of the compute units taken by uncut tiles: 128 tiles of
  // 1 row at 8 stages 14.7 / 18.2, of 64 rows at 6 stages 20.3 / 20.5.  With a longer tile all are cut: 16 x 8 ragged tiles of 1 row and up to 19
  // stages 16.1, with those of up to 6 whole 17.4, of up to 10 19.2 (head_dim 64).
  const int cus = s.cus, i = head_dim / 128;
  const int64_t tiles = (int64_t)B * Hkv * s.rt;
  static constexpr int kLimit[2][3] = {{8, 4, 2}, {4, 3, 2}}, kMore[2][3] = {{8, 8, 4}, {6, 6, 8}};
  s.whole = kLimit[s.staged][i] + (cus > 0 ? (int)(kMore[s.staged][i] * (tiles < cus ? tiles : cus) / cus) : 0);
  s.finer = cus * (s.staged ? 4 : 6);
  return s;
}

// Workgroups per compute unit of a round of equal pieces.  A workgroup is bound by latency, and as many are wanted as fill the memory's
// bandwidth: more only add to what is joined.  For tiles of up to 16 rows that is one with stages of 64 KiB or more (bf16, head_dim
// 128), two with half of that, three with less; for more rows one, and two, all that fit, where row tiles share keys and the matrix units
// are the bound.  Two instead of one: 8192 keys in bf16 13.8 -> 14.4 us, with head_dim 256 19.6 -> 22.7, 131071 keys in e4m3 61.3 -> 57.5;
// 4 x 16 heads of 2521 keys with 32 rows 22.4 -> 24.0, with 256 rows 50.6 -> 44.6.
static int per_cu(const Shape& s, int head_dim, bool f8) {
  if (s.staged || s.nt == 2) return s.rt > 1 ? 2 : 1;
  const int stage = 2 * PA_STAGE * head_dim * (f8 ? 1 : 2);
  return stage >= 65536 ? 1 : stage >= 32768 ? 2 : 3;
}

static int64_t ws_head_floats(int B) { return ((int64_t)2 * B + 63) / 64 * 64; }   // pieces and first slot of every sequence

// Partial results are kept for tiles that are cut only; such a tile has n < 2 * stages / share pieces, and a share is at least the
// `finer`-th part of all stages, so that there are fewer than 2 * finer of them in all; nor are there more than stages.
static int64_t ws_bytes_of(const Shape& s, int B, int Hkv, int max_len, int head_dim) {
  if (s.finer <= 0) return LVAR_ELAUNCH;
  const int64_t stages = ((int64_t)max_len + PA_STAGE - 1) / PA_STAGE;
  if (stages <= s.whole) return 0;   // nothing can be cut
  const int64_t most = (int64_t)B * Hkv * s.rt * stages, slots = most < 2ll * s.finer ? most : 2ll * s.finer;
  return 4 * (ws_head_floats(B) + slots * s.rows * (head_dim + 2));
}
int64_t paged_attn_ws_bytes(int B, int H, int Hkv, int Lq, int max_len, int head_dim) {
  return ws_bytes_of(shape_of(B, H, Hkv, Lq, head_dim), B, Hkv, max_len, head_dim);
}

template <int D, int NT, int W>
static void launch_direct(const PagedAttnParams& p, int grid, hipStream_t s) {
  if (p.cache.k_exp) hipLaunchKernelGGL((paged_attn_kernel<D, NT, true, W>), dim3(grid), dim3(PA_T), 0, s, p);
  else hipLaunchKernelGGL((paged_attn_kernel<D, NT, false, W>), dim3(grid), dim3(PA_T), 0, s, p);
}

template <int D, int NT, int RW, bool F8>
static bool launch_staged(const PagedAttnParams& p, int grid, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int kTiles = 4 * (D == 256 ? 32 : 64) * 2 * D, kOut = PA_WAVES * 16 * (D + 4) * 4, kBytes = kTiles > kOut ? kTiles : kOut;
  if (!ensure_lds_limit((const void*)&paged_tile_kernel<D, NT, RW, F8>, kBytes, done)) return false;
  hipLaunchKernelGGL((paged_tile_kernel<D, NT, RW, F8>), dim3(grid), dim3(PA_T), kBytes, s, p);
  return true;
}
template <int D, int NT, int RW>
static bool launch_staged(const PagedAttnParams& p, int grid, hipStream_t s) {
  return p.cache.k_exp ? launch_staged<D, NT, RW, true>(p, grid, s) : launch_staged<D, NT, RW, false>(p, grid, s);
}

template <int D, int RPB>
static void launch_join(const PagedAttnParams& p, hipStream_t s) {
  hipLaunchKernelGGL((paged_join_kernel<D, RPB>), dim3((p.G * p.Lq + RPB - 1) / RPB, p.cache.kv_heads, p.B), dim3(512), 0, s, p);
}

template <int D>
static int launch_d(const PagedAttnParams& p, const Shape& h, hipStream_t s) {
  const int64_t items = (int64_t)p.B * p.cache.kv_heads * p.rt + (p.ws ? p.finer : 0);
  if (!grid_fits(items + 8, PA_T) || (p.ws && !grid_fits(((int64_t)p.G * p.Lq * D + 2047) / 2048, 512))) return LVAR_EINVAL;
  const int grid = (int)((items + 7) / 8 * 8);
  bool ok = true;
  if constexpr (D == 256) {
    if (!h.staged) launch_direct<D, 1, 2>(p, grid, s);
    else ok = launch_staged<D, 1, 4>(p, grid, s);
  } else {
    if (!h.staged) h.nt == 1 ? launch_direct<D, 1, 3>(p, grid, s) : launch_direct<D, 2, 2>(p, grid, s);
    else ok = h.rw == 2 ? launch_staged<D, 2, 2>(p, grid, s) : launch_staged<D, 2, 4>(p, grid, s);
  }
  if (!ok || hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  if (p.ws) {
    // few rows: all groups along the pieces of one row; many: a group per row
    constexpr int GR = 512 / (D / 4);
    if ((int64_t)p.G * p.Lq * p.cache.kv_heads * p.B <= 4 * h.cus) launch_join<D, 1>(p, s);
    else launch_join<D, GR>(p, s);
    if (hipGetLastError() != hipSuccess) return LVAR_ELAUNCH;
  }
  return LVAR_OK;
}

int launch_paged_attn(PagedAttnParams p, void* workspace, int64_t workspace_bytes, int head_dim, hipStream_t s) {
  const Shape h = shape_of(p.B, p.H, p.cache.kv_heads, p.Lq, head_dim);
  const int64_t need = ws_bytes_of(h, p.B, p.cache.kv_heads, p.max_len, head_dim);
  if (need < 0) return (int)need;
  if (need > 0 && workspace && workspace_bytes >= need) {
    if (((uintptr_t)workspace & 15) != 0) return LVAR_EINVAL;
    p.ws = (float*)workspace;
  }
  p.rt = h.rt;
  p.tile_rows = 16 * h.nt * h.rw;
  // Ragged lengths: two workgroups per compute unit from 4 stages on (tiles of 32 rows and head_dim 128, 16: 8 x 8 tiles of up to 4096 keys 23.7
  // against 25.0 us, 32 x 8 of up to 8000 125 against 116), with head_dim 64 three, which fit, from 16 on (the latter in e4m3, 46 -> 38).
  const int cus = h.cus, per = per_cu(h, head_dim, p.cache.k_exp != nullptr);
  p.target = per * cus;
  p.wide = (per > 2 ? per : 2) * cus;
  p.wider = !h.staged && head_dim == 64 ? 3 * cus : p.wide;
  p.some = (!h.staged && h.nt == 2 && head_dim > 64 ? 16 : 4) * cus;
  p.many = 16 * cus;
  p.most = 64 * cus;
  p.finer = h.finer;
  p.whole = p.ws ? h.whole : 0x7fffffff;   // (no room for partial results: nothing is cut)
  p.slot_rows = h.rows;
  p.ws_head = ws_head_floats(p.B);
  // Pieces of one stage, but of row tiles that are staged only while half of the compute units suffice for them (beyond that the join of the
  // tiles costs more): one sequence of 1024 keys with one new token, 8 of 32 heads, 10.2 -> 8.9 us; 16 heads of 1000 keys with 64 new tokens
  // 16.0 -> 15.3, of 2000 keys 17.6 -> 18.3, 2 x 4 heads of 3000 keys with 256 rows 27.2 -> 31.5.
  p.singles = h.staged ? cus / 2 : 0x7fffffff;
  if (head_dim == 128) return launch_d<128>(p, h, s);
  if (head_dim == 64) return launch_d<64>(p, h, s);
  if (head_dim == 256) return launch_d<256>(p, h, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
