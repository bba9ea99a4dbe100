// What the kernels around the paged key/value cache share: launch parameters, the 8-bit row format, sums inside a row.
//
// The cache holds rows of head_dim keys or values in pages [num_pages, kv_heads, page_size, head_dim], either as bf16 or as
// e4m3 codes with one power of two per row: value = code * 2^(byte - 127), byte the smallest one >= 1 with max|x| <= 448 * 2^(byte - 127).
// A power of two instead of max / 448: scaling and its inverse are exact, a code has 4 significant bits and so every value
// is exact in bf16 -- reading back or feeding the matrix instructions rounds nothing, and the only rounding of a cached
// element is the one to its code.  It costs at most one of e4m3's 15 normal binades at the small end.  (But at the ends of bf16's range: bytes 1 and 2 have
// values below its smallest number's steps, and with byte 247 codes of 256 and more, the code of elements from 1.9375 * 2^127 on, stand for 2^128, an
// infinity there.)
#pragma once
#include "launch.h"

namespace lvar {

struct PagedView {
  uint8_t *k, *v;              // byte pointers (bf16 or e4m3)
  uint8_t *k_exp, *v_exp;      // null: bf16
  int64_t s_page, s_head, s_row;   // bytes
  int64_t e_page, e_head;          // bytes; unit stride along the rows of a page
  const int32_t* table;            // [B, max_pages], row stride table_stride
  int64_t table_stride;
  int num_pages, max_pages, kv_heads;
  int shift;                       // log2(page_size)
};

enum { NORM_NONE = 0, NORM_L2 = 1, NORM_RMS = 2 };
enum { W_NONE = 0, W_HEAD = 1, W_COLUMN = 2 };   // no weight, one factor per head, one per column (of a head or of all)

struct WeightView {
  const void* ptr;
  int64_t s_head;   // elements; 0 = shared by the heads
  int mode;         // W_*
  int bf16;
};

struct NormRopeParams {
  const bf16_t *q, *k, *v;       // v: append only
  int64_t q_sb, q_sh, q_sr, k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;
  bf16_t *oq, *ok;               // contiguous [B,H,L,d], [B,Hkv,L,d]; ok null: k goes into the cache
  WeightView wq, wk;
  int norm;
  float eps, inv_eps;            // inv_eps: set at launch
  const float *cos, *sin;        // [table_rows, rot/2], null: no rotation
  int64_t cs_row;
  int table_rows, rot, interleaved;
  const void* positions;         // int32 or int64, strides in elements; null: the row's own number (plus start[b])
  int64_t pos_sb, pos_sl;
  int pos64;
  int B, H, Hkv, L;
  uint32_t div_mul;              // division by L, set at launch
  int div_s1, div_s2;
  // append
  PagedView cache;
  const int32_t *start, *counts;  // [B]; counts null: L
  int ready;                      // append: k is written as it is, there is no q
  // backward
  const bf16_t *gq, *gk;          // contiguous
  bf16_t *dq, *dk;
  int64_t dq_sb, dq_sh, dq_sr, dk_sb, dk_sh, dk_sr;
  float *pq, *pk;                 // partial weight gradients, null: not wanted, or
  void *dqw, *dkw;                // ... written at once: there is one row of them
  int nblk;
};

// one weight gradient: out[h or 0, column or 0] = sum over the rows of `part` that belong to it
struct WeightGradParams {
  const float* part[2];   // [rows per head, heads, D]: row r of head h at (r * heads + h) * D
  void* out[2];
  int rows[2], heads[2], cols[2], bf16[2];   // cols: 1 (sum over the columns too) or D
  int D;
};

struct KvReadParams {
  PagedView cache;
  bf16_t *k, *v;                  // contiguous [B,Hkv,Lmax,d]
  const int32_t *start, *lengths; // start null: 0
  int B, Lmax;
};

struct PagedAttnParams {
  const bf16_t* q;
  int64_t q_sb, q_sh, q_sr;
  PagedView cache;
  bf16_t* o;                      // contiguous [B,H,Lq,d]
  float *M, *L;                   // [B,H,Lq]
  float* ws;                      // partial results, null: no piece may be cut
  const int32_t *lengths, *counts;
  int B, H, Lq, G, causal;
  int max_len;                    // lengths are clamped to it
  float c;                        // scale * log2(e)
  // set at launch
  int rt, tile_rows;              // row tiles per key/value head, rows of one
  int target, wide, wider, finer, whole;   // pieces of one round, of rounds of more, of several; a call whose tiles have up to this many 128-key stages is not cut
  uint32_t singles;               // up to this many stages in all, pieces may be of one
  uint32_t some, many, most;      // stages in all from which on ragged lengths are cut for `wide`, `wider`, `target` again
  int slot_rows;
  int64_t ws_head;                // floats ahead of the partial results
};

constexpr int NB_HC = 2;   // heads of a workgroup of the norm's backward pass

// A launch has at most 2^32 - 1 threads along x.
inline bool grid_fits(int64_t workgroups, int threads) { return workgroups * threads <= 0xffffffffll; }

int launch_norm_rope(NormRopeParams p, int head_dim, bool append, hipStream_t s);
int norm_rope_bwd_blocks(int B, int H, int Hkv, int L, int head_dim, bool alone);
int launch_norm_rope_bwd(NormRopeParams p, int head_dim, hipStream_t s);
int launch_weight_grad(const WeightGradParams& w, hipStream_t s);
int launch_kv_read(const KvReadParams& p, int head_dim, hipStream_t s);
int64_t paged_attn_ws_bytes(int B, int H, int Hkv, int Lq, int max_len, int head_dim);
int launch_paged_attn(PagedAttnParams p, void* workspace, int64_t workspace_bytes, int head_dim, hipStream_t s);

template <int CTRL>
__device__ __forceinline__ int dpp_mov(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }

// Butterfly over aligned groups of LANES lanes (2 .. 32): quad swaps, mirrors inside 8 and 16, rows of 16.  Every step adds the same
// two partial results in every lane that takes part, so all lanes of a group end with the same bits.
template <int LANES, class F>
__device__ __forceinline__ int row_fold(int x, F f) {
  x = f(x, dpp_mov<0xB1>(x));                               // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) x = f(x, dpp_mov<0x4E>(x));     // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) x = f(x, dpp_mov<0x141>(x));    // row_half_mirror
  if constexpr (LANES >= 16) x = f(x, dpp_mov<0x140>(x));   // row_mirror
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f((int)r[0], (int)r[1]);
  }
  return x;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  return __builtin_bit_cast(float, row_fold<LANES>(__builtin_bit_cast(int, x), [](int a, int b) {
    return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
  }));
}
template <int LANES>
__device__ __forceinline__ uint32_t row_umax(uint32_t x) {
  return (uint32_t)row_fold<LANES>((int)x, [](int a, int b) { return (int)((uint32_t)a > (uint32_t)b ? (uint32_t)a : (uint32_t)b); });
}

__device__ __forceinline__ void unpack8(u32x4 u, float* f) {
#pragma unroll
  for (int e = 0; e < 4; e++) { f[2 * e] = bf16_lo(u[e]); f[2 * e + 1] = bf16_hi(u[e]); }
}
__device__ __forceinline__ u32x4 pack8u(const float* f) {
  return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
}

// Bits of |x| of a finite x, 0 for infinities and NaN (tested on the bits: the float comparisons may assume that there are none).
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return a < 0x7f800000u ? a : 0u;
}

// Exponent byte of a row whose largest finite magnitude has these bits: 448 = 1.75 * 2^8, so the exponent rises by one where the fraction is above .75.
__device__ __forceinline__ uint32_t exp_byte(uint32_t top) {
  const int e = (int)((top + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(e > 1 ? e : 1);
}
__device__ __forceinline__ float exp_value(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
__device__ __forceinline__ float exp_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }

// Codes of 8 values, round to nearest even; infinities and NaN become NaN (e4m3 has no infinity).
__device__ __forceinline__ u32x2 codes8(const float* f, uint32_t byte) {
  const float inv = exp_inverse(byte);
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h] * inv, f[4 * h + 1] * inv, 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2] * inv, f[4 * h + 3] * inv, u, true);
    uint32_t w = (uint32_t)u;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if ((__builtin_bit_cast(uint32_t, f[4 * h + e]) & 0x7f800000u) == 0x7f800000u) w |= 0x7fu << (8 * e);
    r[h] = w;
  }
  return r;
}

// bf16 values of 8 codes (exact)
__device__ __forceinline__ u32x4 values8(u32x2 c, float scale) {
  u32x4 r;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
    r[2 * h] = pack_bf16(a[0] * scale, a[1] * scale);
    r[2 * h + 1] = pack_bf16(b[0] * scale, b[1] * scale);
  }
  return r;
}

// Place of token `pos` of sequence b: false where the table does not reach it or names no page of the pool.
__device__ __forceinline__ bool find_row(const PagedView& c, int b, int64_t pos, int& page, int& slot) {
  page = 0; slot = 0;
  const int64_t at = pos >> c.shift;
  if (pos < 0 || at >= c.max_pages) return false;
  const int pg = c.table[b * c.table_stride + at];
  if (pg < 0 || pg >= c.num_pages) return false;
  page = pg;
  slot = (int)(pos & ((1ll << c.shift) - 1));
  return true;
}

}  // namespace lvar
