// What the kernels of the attention over packed sequences share: launch parameters, which tile a workgroup takes, filling a tile into LDS.
//
// Sequence b of a batch has queries offsets[b] .. offsets[b+1]-1 and keys k_offsets[b] .. k_offsets[b+1]-1 of the packed tensors
// [heads, tokens, d].  Row i of n queries over m keys sees keys j < m - n + i + 1 (causal) or j < m.
#pragma once
#include "attn_tile.h"
#include "launch.h"

namespace lvar {

struct PackedParams {
  const bf16_t *q, *k, *v;
  int64_t q_sh, q_sr, k_sh, k_sr, v_sh, v_sr;
  bf16_t* o;                        // [H,T,d], strides o_sh, o_sr
  int64_t o_sh, o_sr;
  float *M, *L;                     // [H,T]
  const int32_t *q_off, *k_off;     // [B+1]
  int B, T, Tk, H, Hkv, G, causal;
  float c, scale;                   // c = scale * log2(e)
  // backward
  const bf16_t* g;                  // gradient of o
  int64_t g_sh, g_sr;
  bf16_t *dq, *dk, *dv;             // null: not wanted
  int64_t dq_sh, dq_sr, dk_sh, dk_sr, dv_sh, dv_sr;
  int slots;                        // set at launch: places for query tiles, see find_tile
  int shares;                       // set at launch: workgroups that share the keys of a query tile, or the query rows of a key tile
  float* parts;                     // their sums: [shares][H][T][D] of o or dq, [shares][dk, dv][Hkv][Tk][D]
  float* part_stats;                // forward: [shares][H][T][3] what their P refers to, its sum, the maximum
  int settle;                       // set at launch: deltas of rows with few keys are corrected, see packed_dq_kernel
  float* stats;                     // [H,2,T]: -(M + log2 L) / c (-inf: the row sees nothing), and -sum(do * o)
};

int64_t packed_fwd_bytes(const PackedParams& p, int head_dim);
int launch_packed_fwd(PackedParams p, void* workspace, int head_dim, hipStream_t s);
int64_t packed_bwd_bytes(const PackedParams& p, int head_dim);
int launch_packed_bwd(PackedParams p, void* workspace, int head_dim, hipStream_t s);

// Tiles of R rows of T packed rows in B sequences: the ranges between sequence borders, one ahead of the first sequence and one
// behind the last included, have at most these many.
inline int64_t packed_slots(int T, int B, int R) { return (int64_t)T / R + B + 2; }

// Workgroups that share the keys of a query tile of 128 rows, where query tiles alone leave compute units idle (few rows over many keys, few heads): as
// many as fill the waves that a SIMD holds, twice that if causal, where the last tile has twice the work of the mean one.  None gets fewer than
// SHARE_TILES tiles of the mean sequence (lengths are on the device: one long sequence among many short ones is not shared): parts cost a launch and
// 8 bytes of traffic per element, about what 9 us of products are worth.  Against one workgroup per tile, forward / dq, the sum of the parts included: 64 rows of 8 heads of 128 over 8192 keys 93 -> 22 / 144 -> 28 us; 16384 rows
// of one head, causal 198 -> 91 / 302 -> 126 us; 9360 rows of 4 heads of 64, causal 95 -> 71 / 126 -> 90 us.  With shares of 4 tiles 2048 rows of 16 heads of
// 128, causal lost: 35 -> 44 / 51 -> 55 us.
inline int query_shares(const PackedParams& p, int waves_per_simd) {
  constexpr int SHARE_TILES = 12;
  const int64_t groups = ((int64_t)p.T / 128 + p.B) * p.H, slots = (int64_t)device_cus() * waves_per_simd * (p.causal ? 2 : 1);
  const int64_t most = (int64_t)p.Tk / p.B / 64 / (p.causal ? 2 : 1) / SHARE_TILES, want = slots / (groups > 0 ? groups : 1);
  const int64_t n = want < most ? want : most;
  return n < 2 ? 1 : n > 32 ? 32 : (int)n;
}

#if defined(__HIP_DEVICE_COMPILE__)

// Tiles t0 .. t0 + T - 1 of a share of T_all
struct Share { int t0, T; };
__device__ __forceinline__ Share share_of(int T_all, int share, int shares) {
  const int t0 = (int)((int64_t)T_all * share / shares);
  return {t0, (int)((int64_t)T_all * (share + 1) / shares) - t0};
}

// Sum over the 64 lanes, the same in all of them
__device__ __forceinline__ int wave_sum(int x) {
  auto add = [](int v, auto ctrl) { return v + __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, 0xf, 0xf, true); };
  x = add(x, std::integral_constant<int, 0xB1>{});    // quad_perm [1,0,3,2]
  x = add(x, std::integral_constant<int, 0x4E>{});    // quad_perm [2,3,0,1]
  x = add(x, std::integral_constant<int, 0x141>{});   // row_half_mirror
  x = add(x, std::integral_constant<int, 0x140>{});   // row_mirror
  return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48);
}

struct PackedTile {
  int first, n;               // the sequence's first row and how many it has
  int row0;                   // first row of the tile within it
  int other_first, other_n;   // its rows on the other side (keys of a query tile, queries of a key tile); none for rows of no sequence
};

// Border v of the B + 3 borders of T rows: 0, the offsets, T.  (Offsets out of range, a caller's mistake, stay in it.)
__device__ __forceinline__ int packed_border(const int32_t* off, int B, int T, int v) {
  if (v <= 0) return 0;
  return v > B + 1 ? T : max(0, min(off[v - 1], T));
}

// The range and tile of place `slot`, and the sequence's rows on the other side.  Range v takes the places from floor(border(v) / R) + v on: a range of
// n rows starting anywhere has at most floor((border + n) / R) - floor(border / R) + 1 tiles, so its places suffice, and which range a
// place belongs to is found among the borders without knowing the lengths in between: 64 candidates per step, and with up to 62 sequences in
// one round trip to memory.  False: a place without a tile.
//
// `levels` (up to 62 sequences, a lane each; beyond, the order of the places is kept, and what that costs there is not measured): of a causal launch
// over key tiles those of a range differ in work, the first having the most
// rows behind it, and the launch would end on whichever long one comes late: place by place the tiles with the most behind
// them, of all ranges.  (12 sequences of up to 2047 tokens, 8 x 4 heads, in the kernel of that time:
// 492 -> 404 us.  Query tiles, four times as many and each shorter: 3 % less for these, 2 % more for 16 prompts of up to 4096.)
template <int R>
__device__ __forceinline__ bool find_tile(const int32_t* off, int T, const int32_t* other, int other_T, int B, int slot, bool levels, PackedTile& t) {
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  int v;
  if (B + 2 <= 64) {
    const int first = packed_border(off, B, T, lane), next = packed_border(off, B, T, lane + 1);
    const int o_first = packed_border(other, B, other_T, lane), o_next = packed_border(other, B, other_T, lane + 1);
    const bool range = lane < B + 2;
    if (levels) {
      const int tiles = range ? (max(0, next - first) + R - 1) / R : 0;
      auto tiles_from = [&](int level) { return wave_sum(max(0, tiles - level)); };   // on levels level + 1 and up
      if (slot >= tiles_from(0)) return false;
      int lo = 0, hi = (T + R - 1) / R;                                               // tiles_from(hi) <= slot < tiles_from(lo)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles_from(mid) <= slot) hi = mid; else lo = mid;
      }
      const int rank = slot - tiles_from(hi);   // among the ranges with a tile on level hi
      const uint64_t mine = __builtin_amdgcn_ballot_w64(tiles >= hi);
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mine >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mine, 0));
      v = __builtin_ctzll(__builtin_amdgcn_ballot_w64(tiles >= hi && before == rank));
      t.row0 = (__builtin_amdgcn_readlane(tiles, v) - hi) * R;
    } else {
      const uint64_t mine = __builtin_amdgcn_ballot_w64(range && first / R + lane <= slot);
      v = mine ? 63 - __builtin_clzll(mine) : 0;
      t.row0 = (slot - (__builtin_amdgcn_readlane(first, v) / R + v)) * R;
    }
    t.first = __builtin_amdgcn_readlane(first, v);
    t.n = __builtin_amdgcn_readlane(next, v) - t.first;
    t.other_first = __builtin_amdgcn_readlane(o_first, v);
    t.other_n = __builtin_amdgcn_readlane(o_next, v) - t.other_first;
  } else {
    v = 0;
    int n = B + 2;
    while (n > 1) {
      const int step = (n + 63) >> 6, at = v + lane * step;
      const bool in = lane * step < n;
      const int e = packed_border(off, B, T, in ? at : 0);
      const uint64_t mine = __builtin_amdgcn_ballot_w64(in && e / R + at <= slot);
      const int k = mine ? 63 - __builtin_clzll(mine) : 0;
      v += k * step;
      n = min(step, n - k * step);
    }
    v = __builtin_amdgcn_readfirstlane(v);
    const int two = v + (lane & 1);
    const int e = packed_border(off, B, T, two), o = packed_border(other, B, other_T, two);
    t.first = __builtin_amdgcn_readlane(e, 0);
    t.n = __builtin_amdgcn_readlane(e, 1) - t.first;
    t.row0 = (slot - (t.first / R + v)) * R;
    t.other_first = __builtin_amdgcn_readlane(o, 0);
    t.other_n = __builtin_amdgcn_readlane(o, 1) - t.other_first;
  }
  if (v == 0 || v > B) t.other_n = 0;
  t.other_n = max(0, t.other_n);
  return t.row0 >= 0 && t.row0 < t.n;
}

// The sequence of row `row` and its rows on both sides; none on the other side for rows of no sequence.
__device__ __forceinline__ void find_row(const int32_t* off, int T, const int32_t* other, int other_T, int B, int row, PackedTile& t) {
  const int lane = __builtin_amdgcn_workitem_id_x() & 63;
  int v = 0, n = B + 2;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = v + lane * step;
    const bool in = lane * step < n;
    const uint64_t mine = __builtin_amdgcn_ballot_w64(in && packed_border(off, B, T, in ? at : 0) <= row);
    const int k = mine ? 63 - __builtin_clzll(mine) : 0;
    v += k * step;
    n = min(step, n - k * step);
  }
  v = __builtin_amdgcn_readfirstlane(v);
  t.first = packed_border(off, B, T, v);
  t.n = packed_border(off, B, T, v + 1) - t.first;
  t.row0 = row - t.first;
  t.other_first = packed_border(other, B, other_T, v);
  t.other_n = v == 0 || v > B ? 0 : max(0, packed_border(other, B, other_T, v + 1) - t.other_first);
}

// Rows of D bf16 in LDS, unpadded (an LDS fill writes 1 KiB of consecutive bytes), the 16-byte chunks of a row moved by an XOR that suits both
// ways of reading: 16 consecutive rows, one chunk each (ds_read_b128), lie on all banks, since the XOR is another one for every
// row of 16 (of 8 pairs of rows at D = 64); and 4 consecutive rows, one 64-byte segment each (transposing reads), too, since its upper
// bits, which move segments, are the lower bits of the row.
template <int D>
struct PackedLds {
  static constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 1024 / ROWB, NI = 64 / RPI, TILE = 64 * ROWB;
  __device__ static __forceinline__ int swz(int row) {
    return D >= 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  }
  int row_at, tr_at;   // byte offsets of this lane's reads
  __device__ __forceinline__ PackedLds(int lane) {
    const int hh = lane >> 5, r = lane & 31, sq = (lane & 15) >> 2, sm = lane & 3;
    row_at = r * ROWB + ((hh ^ swz(r)) << 4);
    tr_at = (4 * hh + sq) * ROWB + (((((lane >> 4) & 1) << 1 | (sm >> 1)) ^ swz(4 * hh + sq)) << 4) + (sm & 1) * 8;
  }
  // A operand of rows 32 sub .. +31, columns 16 ks .. +15
  __device__ __forceinline__ bf16x8 rows(const char* buf, int sub, int ks) const {
    return *(const bf16x8*)(buf + (row_at ^ (ks << 5)) + sub * 32 * ROWB);
  }
  // A operand of columns 32 m .. +31 (as rows) over rows 16 kb .. +15, in the order in which accumulators hold them
  __device__ __forceinline__ bf16x8 columns(const char* buf, int kb, int m) const {
    const char* a = buf + kb * 16 * ROWB;
    const int at = tr_at ^ (m << 6);
    const bf16x4 lo = lds_read_tr(a + at), hi = lds_read_tr(a + (at ^ 32) + 8 * ROWB);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// The same operands from LDS byte addresses that hold the lane's own offset (row_at, tr_at) already, on buffers aligned to 512 bytes: what differs per
// operand is an XOR or part of the instruction, and nothing is kept in registers for it.
template <int D>
struct PackedOperands {
  static __device__ __forceinline__ bf16x8 rows(uint32_t at, int ks) { return *(LVAR_LDS const bf16x8*)(uintptr_t)(at ^ (ks << 5)); }
  static __device__ __forceinline__ bf16x8 columns(uint32_t at, int kb, int m) {
    const uint32_t lo = at ^ (m << 6), hi = at ^ (m << 6) ^ 32;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LVAR_LDS bf16x4*)(uintptr_t)(lo + kb * 32 * D));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LVAR_LDS bf16x4*)(uintptr_t)(hi + kb * 32 * D + 16 * D));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Raw buffer descriptor of `bytes` from base on (below 2^31, checked on the host): what lies beyond reads as zeros.
__device__ __forceinline__ i32x4 packed_rsrc(const void* base, int bytes) {
  const uint64_t a = (uint64_t)base;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)((a >> 32) & 0xffffu)),
               __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// ... of n rows
__device__ __forceinline__ i32x4 packed_rsrc(const bf16_t* base, int n, int row_bytes, int stride_bytes) {
  return packed_rsrc(base, n > 0 ? (n - 1) * stride_bytes + row_bytes : 0);
}

// One of the fills of rows row0 .. row0 + 63 into LDS at byte address dst: the s-th of the NI / NW that a wave issues.  Inline assembly, so that
// the compiler does not make LDS reads of other buffers wait for it; wait_fills() before the barrier does.
template <int D, int NW>
__device__ __forceinline__ void fill_slot(const i32x4& rsrc, int srb, int row0, uint32_t dst, int wave, int lane, int s) {
  using S = PackedLds<D>;
  static_assert(S::NI % NW == 0, "every wave issues as many fills");
  // the XOR has a period of 16 rows: fills whose rows are whole periods apart share the lane's offset
  constexpr int PER = NW * S::RPI >= 16 ? 1 : 16 / (NW * S::RPI);
  const int lrow = lane / S::CPR, lcs = lane % S::CPR;
  const int trow = (wave + (s % PER) * NW) * S::RPI + lrow;
  const int voff = trow * srb + ((lcs ^ S::swz(trow)) << 4);
  const int soff = (row0 + (s / PER) * PER * NW * S::RPI) * srb;
  const uint32_t m0v = dst + (wave + s * NW) * 1024;
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(m0v), "v"(voff), "s"(rsrc), "s"(soff)
      : "memory");
}
// The NR / RPI / NW fills of a wave for NR rows
template <int D, int NW, int NR>
__device__ __forceinline__ void fill_rows(const i32x4& rsrc, int srb, int row0, uint32_t dst, int wave, int lane) {
  static_assert(NR / PackedLds<D>::RPI % NW == 0, "every wave issues as many fills");
#pragma unroll
  for (int s = 0; s < NR / PackedLds<D>::RPI / NW; s++) fill_slot<D, NW>(rsrc, srb, row0, dst, wave, lane, s);
}
template <int D, int NW>
__device__ __forceinline__ void fill_tile(const i32x4& rsrc, int srb, int row0, uint32_t dst, int wave, int lane) {
#pragma unroll
  for (int s = 0; s < PackedLds<D>::NI / NW; s++) fill_slot<D, NW>(rsrc, srb, row0, dst, wave, lane, s);
}

// Head of place j of H: with a multiple of 8 heads, those of an XCD (workgroups are dealt to the 8 in turn) are neighbours, which share keys and values.
__device__ __forceinline__ int packed_head(int j, int H) { return (H & 7) == 0 ? (j & 7) * (H >> 3) + (j >> 3) : j; }

// The bits of x, which the compiler cannot trace back to a float: with -fno-honor-nans it takes a test of them for one of a number.
__device__ __forceinline__ uint32_t bits_of(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  asm("" : "+v"(u));
  return u;
}
// Is x infinite or NaN?
__device__ __forceinline__ bool not_finite(float x) { return (bits_of(x) & 0x7f800000u) == 0x7f800000u; }

// The transposed accumulators of a wave, 32 rows of D columns, as bf16 rows: through LDS (32 * (2 D + 16) bytes at `buf`, this wave's
// own), so that rows are stored in 16-byte pieces.  rows < n are stored.
template <int D, int MT>
__device__ __forceinline__ void store_rows(char* buf, const f32x16 (&acc)[MT], float factor, bf16_t* to, int64_t stride, int n, int lane) {
  static_assert(MT * 32 == D, "all columns");
  constexpr int STR = D * 2 + 16, CPR = D / 8;
  const int hh = lane >> 5, r = lane & 31;
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int a = 0; a < 4; a++) {
      const u32x2 pk = {pack_bf16(acc[m][4 * a] * factor, acc[m][4 * a + 1] * factor), pack_bf16(acc[m][4 * a + 2] * factor, acc[m][4 * a + 3] * factor)};
      *(u32x2*)(buf + r * STR + (m * 32 + 8 * a + 4 * hh) * 2) = pk;
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 32 * CPR / 64; i++) {
    const int at = lane + i * 64, row = at / CPR, chunk = at - row * CPR;
    const u32x4 x = *(const u32x4*)(buf + row * STR + chunk * 16);
    if (row < n) *(u32x4*)(to + row * stride + chunk * 8) = x;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The same sums as they are, fp32 rows of D one behind the other, half of the columns at a time through the same bytes of LDS.  (Straight from the
// accumulators, 16 bytes of each row per instruction, the stores of three shares of 2048 rows of 16 heads of 128 took longer than their products.)
template <int D, int MT>
__device__ __forceinline__ void store_part(char* buf, const f32x16 (&acc)[MT], float* to, int n, int lane) {
  static_assert(MT * 32 == D, "all columns");
  constexpr int STR = D * 2 + 16, CPR = D / 8;   // bytes of half a row, 16-byte pieces
  const int hh = lane >> 5, r = lane & 31;
#pragma unroll
  for (int half = 0; half < 2; half++) {
#pragma unroll
    for (int m = 0; m < MT / 2; m++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        const f32x16& x = acc[half * (MT / 2) + m];
        *(f32x4*)(buf + r * STR + (m * 32 + 8 * a + 4 * hh) * 4) = f32x4{x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]};
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 32 * CPR / 64; i++) {
      const int at = lane + i * 64, row = at / CPR, chunk = at - row * CPR;
      const f32x4 x = *(const f32x4*)(buf + row * STR + chunk * 16);
      if (row < n) *(f32x4*)(to + row * D + half * (D / 2) + chunk * 4) = x;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

#endif  // __HIP_DEVICE_COMPILE__

}  // namespace lvar
