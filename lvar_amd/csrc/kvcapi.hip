// extern "C" entry points of the norms, the paged cache and the attention over it: argument checks and parameter packing.
#include <cmath>
#include "kvcache.h"

using namespace lvar;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMostTokens = 1ll << 30;   // B * L, table reach: token numbers and tile origins stay within 31 bits

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool rows_ok(const lvar_tensor_t& t) {
  return t.ptr && aligned(t.ptr, 16) && t.stride_b % 8 == 0 && t.stride_h % 8 == 0 && t.stride_row % 8 == 0;
}

int sizes_ok(int B, int H, int kv_heads, int L) {
  if (B <= 0 || L <= 0 || kv_heads <= 0 || H <= 0 || H % kv_heads != 0) return LVAR_EINVAL;
  // grid axes: batch and heads on y and z (the x axis is checked where its workgroups are counted)
  if (B > 65535 || H > 16384 || (int64_t)B * L > kMostTokens) return LVAR_EINVAL;
  return LVAR_OK;
}

bool norm_head_dim(int d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }
bool cache_head_dim(int d) { return d == 64 || d == 128 || d == 256; }

bool weight_ok(const lvar_weight_t& w, WeightView& v) {
  v = {};
  if (!w.ptr) return true;
  if ((w.dtype != 0 && w.dtype != 1) || (w.stride_col != 0 && w.stride_col != 1)) return false;
  if (w.stride_col == 1 && (!aligned(w.ptr, 16) || w.stride_head % 8 != 0)) return false;
  if (!aligned(w.ptr, w.dtype ? 2 : 4)) return false;
  v.ptr = w.ptr; v.s_head = w.stride_head; v.bf16 = w.dtype;
  v.mode = w.stride_col ? W_COLUMN : W_HEAD;
  return true;
}

int fill_how(NormRopeParams& p, const lvar_norm_rope_t& how, int head_dim) {
  if (how.norm < LVAR_NORM_NONE || how.norm > LVAR_NORM_RMS || !(how.eps == 0.f || std::isnormal(how.eps)) || how.eps < 0.f) return LVAR_EINVAL;
  if (!weight_ok(how.q_weight, p.wq) || !weight_ok(how.k_weight, p.wk)) return LVAR_EINVAL;
  p.norm = how.norm; p.eps = how.eps;
  if (!how.cos != !how.sin) return LVAR_EINVAL;
  if (how.cos) {
    if (how.rot_dim <= 0 || how.rot_dim > head_dim || how.table_rows <= 0) return LVAR_EINVAL;
    if (how.rot_dim % 16 != 0) return LVAR_EUNSUPPORTED;
    if (!aligned(how.cos, 16) || !aligned(how.sin, 16) || how.table_stride % 4 != 0 || how.table_stride < 0) return LVAR_EINVAL;
    if (how.positions && !aligned(how.positions, how.positions64 ? 8 : 4)) return LVAR_EINVAL;
    p.cos = how.cos; p.sin = how.sin; p.cs_row = how.table_stride; p.table_rows = how.table_rows; p.rot = how.rot_dim;
    p.interleaved = how.interleaved ? 1 : 0;
    p.positions = how.positions; p.pos_sb = how.pos_stride_b; p.pos_sl = how.pos_stride_row; p.pos64 = how.positions64 ? 1 : 0;
  }
  return LVAR_OK;
}

void fill_qk(NormRopeParams& p, const lvar_tensor_t& q, const lvar_tensor_t& k, int B, int H, int kv_heads, int L) {
  p.q = (const bf16_t*)q.ptr; p.q_sb = q.stride_b; p.q_sh = q.stride_h; p.q_sr = q.stride_row;
  p.k = (const bf16_t*)k.ptr; p.k_sb = k.stride_b; p.k_sh = k.stride_h; p.k_sr = k.stride_row;
  p.B = B; p.H = H; p.Hkv = kv_heads; p.L = L;
}

int fill_cache(PagedView& v, const lvar_paged_cache_t& c) {
  if (!c.k || !c.v || !c.page_table || !c.k_exp != !c.v_exp || c.num_pages <= 0 || c.max_pages <= 0 || c.kv_heads <= 0) return LVAR_EINVAL;
  if (c.page_size <= 0 || c.table_stride < 0) return LVAR_EINVAL;
  if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)) != 0 || !cache_head_dim(c.head_dim)) return LVAR_EUNSUPPORTED;
  const int64_t size = c.k_exp ? 1 : 2;   // bytes of an element
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || c.stride_page < 0 || c.stride_head < 0 || c.stride_row < c.head_dim ||
      c.stride_page * size % 16 != 0 || c.stride_head * size % 16 != 0 || c.stride_row * size % 16 != 0)
    return LVAR_EINVAL;
  if (c.stride_row * size >= 1ll << 27) return LVAR_EINVAL;   // 16 rows within 32 bits
  if (c.k_exp && (!aligned(c.k_exp, 4) || !aligned(c.v_exp, 4) || c.exp_stride_page % 4 != 0 || c.exp_stride_head % 4 != 0 ||
                  c.exp_stride_page < 0 || c.exp_stride_head < 0))
    return LVAR_EINVAL;
  if (!aligned(c.page_table, 4) || (int64_t)c.max_pages * c.page_size > kMostTokens) return LVAR_EINVAL;
  v.k = (uint8_t*)c.k; v.v = (uint8_t*)c.v; v.k_exp = c.k_exp; v.v_exp = c.v_exp;
  v.s_page = c.stride_page * size; v.s_head = c.stride_head * size; v.s_row = c.stride_row * size;
  v.e_page = c.exp_stride_page; v.e_head = c.exp_stride_head;
  v.table = c.page_table; v.table_stride = c.table_stride;
  v.num_pages = c.num_pages; v.max_pages = c.max_pages; v.kv_heads = c.kv_heads;
  v.shift = __builtin_ctz((unsigned)c.page_size);
  return LVAR_OK;
}

// partial rows of a weight gradient
int grad_rows(const WeightView& w, int heads, int nblk) { return w.s_head == 0 ? nblk * ((heads + NB_HC - 1) / NB_HC) : nblk; }
int64_t grad_floats(int heads, int nblk, int d) { return (int64_t)nblk * heads * d; }   // (the larger of the two forms)

}  // namespace

extern "C" {

int lvar_qk_norm_rope_fwd(lvar_tensor_t q, lvar_tensor_t k, lvar_norm_rope_t how, void* oq, void* ok, int B, int H, int kv_heads,
                          int L, int head_dim, void* stream) {
  int st = sizes_ok(B, H, kv_heads, L);
  if (st != LVAR_OK) return st;
  if (!rows_ok(q) || !rows_ok(k) || !oq || !ok || !aligned(oq, 16) || !aligned(ok, 16)) return LVAR_EINVAL;
  if (!norm_head_dim(head_dim)) return LVAR_EUNSUPPORTED;
  NormRopeParams p{};
  fill_qk(p, q, k, B, H, kv_heads, L);
  if ((st = fill_how(p, how, head_dim)) != LVAR_OK) return st;
  p.oq = (bf16_t*)oq; p.ok = (bf16_t*)ok;
  return launch_norm_rope(p, head_dim, false, (hipStream_t)stream);
}

int64_t lvar_qk_norm_rope_bwd_scratch_bytes(int B, int H, int kv_heads, int L, int head_dim) {
  const int st = sizes_ok(B, H, kv_heads, L);
  if (st != LVAR_OK) return st;
  if (!norm_head_dim(head_dim)) return LVAR_EUNSUPPORTED;
  const int nblk = norm_rope_bwd_blocks(B, H, kv_heads, L, head_dim, false);
  if (nblk <= 0) return LVAR_ELAUNCH;
  return 4 * grad_floats(H + kv_heads, nblk, head_dim);
}

int lvar_qk_norm_rope_bwd(lvar_tensor_t q, lvar_tensor_t k, lvar_norm_rope_t how, const void* gq, const void* gk, lvar_tensor_t dq,
                          lvar_tensor_t dk, void* dqw, void* dkw, void* scratch, int64_t scratch_bytes, int B, int H,
                          int kv_heads, int L, int head_dim, void* stream) {
  int st = sizes_ok(B, H, kv_heads, L);
  if (st != LVAR_OK) return st;
  if (!rows_ok(q) || !rows_ok(k) || !rows_ok(dq) || !rows_ok(dk) || !gq || !gk || !aligned(gq, 16) || !aligned(gk, 16)) return LVAR_EINVAL;
  if ((dqw && !how.q_weight.ptr) || (dkw && !how.k_weight.ptr)) return LVAR_EINVAL;
  if (!norm_head_dim(head_dim)) return LVAR_EUNSUPPORTED;
  NormRopeParams p{};
  fill_qk(p, q, k, B, H, kv_heads, L);
  if ((st = fill_how(p, how, head_dim)) != LVAR_OK) return st;
  p.gq = (const bf16_t*)gq; p.gk = (const bf16_t*)gk;
  p.dq = (bf16_t*)dq.ptr; p.dq_sb = dq.stride_b; p.dq_sh = dq.stride_h; p.dq_sr = dq.stride_row;
  p.dk = (bf16_t*)dk.ptr; p.dk_sb = dk.stride_b; p.dk_sh = dk.stride_h; p.dk_sr = dk.stride_row;
  // (a weight whose heads do not differ in memory gets one gradient for all of them)
  if (dqw || dkw) {
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < lvar_qk_norm_rope_bwd_scratch_bytes(B, H, kv_heads, L, head_dim)) return LVAR_EINVAL;
  }
  const WeightView* wv[2] = {&p.wq, &p.wk};
  void* out[2] = {dqw, dkw};
  const int heads[2] = {H, kv_heads};
  bool alone = dqw || dkw;
  for (int i = 0; i < 2; i++) alone = alone && !(out[i] && wv[i]->s_head == 0 && heads[i] > NB_HC);
  p.nblk = norm_rope_bwd_blocks(B, H, kv_heads, L, head_dim, alone);
  if (p.nblk <= 0) return LVAR_ELAUNCH;
  float* parts[2] = {(float*)scratch, (float*)scratch + grad_floats(H, p.nblk, head_dim)};
  WeightGradParams w{};
  w.D = head_dim;
  bool rest = false;
  for (int i = 0; i < 2; i++) {
    if (!out[i]) continue;
    const int rows = grad_rows(*wv[i], heads[i], p.nblk);
    if (rows == 1) {
      (i ? p.dkw : p.dqw) = out[i];
      continue;
    }
    rest = true;
    (i ? p.pk : p.pq) = parts[i];
    w.out[i] = out[i]; w.part[i] = parts[i];
    w.heads[i] = wv[i]->s_head == 0 ? 1 : heads[i];
    w.rows[i] = rows;
    w.cols[i] = wv[i]->mode == W_COLUMN ? head_dim : 1;
    w.bf16[i] = wv[i]->bf16;
  }
  if ((st = launch_norm_rope_bwd(p, head_dim, (hipStream_t)stream)) != LVAR_OK || !rest) return st;
  return launch_weight_grad(w, (hipStream_t)stream);
}

int lvar_kv_cache_append(lvar_tensor_t q, lvar_tensor_t k, lvar_tensor_t v, const lvar_norm_rope_t* how, void* oq, lvar_paged_cache_t cache,
                         const int32_t* start, const int32_t* counts, int B, int H, int L, void* stream) {
  NormRopeParams p{};
  int st = fill_cache(p.cache, cache);
  if (st != LVAR_OK) return st;
  if (!how) H = cache.kv_heads;
  if ((st = sizes_ok(B, H, cache.kv_heads, L)) != LVAR_OK) return st;
  if (!rows_ok(k) || !rows_ok(v) || !start || !aligned(start, 4) || !aligned(counts, 4) || !how != !oq) return LVAR_EINVAL;
  if (how && (!rows_ok(q) || !aligned(oq, 16))) return LVAR_EINVAL;
  fill_qk(p, q, k, B, H, cache.kv_heads, L);
  p.v = (const bf16_t*)v.ptr; p.v_sb = v.stride_b; p.v_sh = v.stride_h; p.v_sr = v.stride_row;
  if (how && (st = fill_how(p, *how, cache.head_dim)) != LVAR_OK) return st;
  p.ready = how ? 0 : 1;
  p.oq = (bf16_t*)oq;
  p.start = start; p.counts = counts;
  return launch_norm_rope(p, cache.head_dim, true, (hipStream_t)stream);
}

int lvar_kv_cache_read(lvar_paged_cache_t cache, const int32_t* start, const int32_t* lengths, void* k, void* v, int B, int max_len,
                       void* stream) {
  KvReadParams p{};
  int st = fill_cache(p.cache, cache);
  if (st != LVAR_OK) return st;
  if ((st = sizes_ok(B, cache.kv_heads, cache.kv_heads, max_len)) != LVAR_OK) return st;
  if (!k || !v || !aligned(k, 16) || !aligned(v, 16) || !lengths || !aligned(lengths, 4) || !aligned(start, 4)) return LVAR_EINVAL;
  p.k = (bf16_t*)k; p.v = (bf16_t*)v; p.start = start; p.lengths = lengths; p.B = B; p.Lmax = max_len;
  return launch_kv_read(p, cache.head_dim, (hipStream_t)stream);
}

int64_t lvar_paged_attn_workspace_bytes(int B, int H, int kv_heads, int Lq, int max_len, int head_dim) {
  const int st = sizes_ok(B, H, kv_heads, Lq);
  if (st != LVAR_OK) return st;
  if (max_len < 0) return LVAR_EINVAL;
  if (!cache_head_dim(head_dim)) return LVAR_EUNSUPPORTED;
  return paged_attn_ws_bytes(B, H, kv_heads, Lq, max_len, head_dim);
}

int lvar_paged_attn_fwd(lvar_tensor_t q, lvar_paged_cache_t cache, const int32_t* lengths, const int32_t* counts, void* o, float* M,
                        float* L, void* workspace, int64_t workspace_bytes, int B, int H, int Lq, int max_len, int causal,
                        float scale, void* stream) {
  PagedAttnParams p{};
  int st = fill_cache(p.cache, cache);
  if (st != LVAR_OK) return st;
  if ((st = sizes_ok(B, H, cache.kv_heads, Lq)) != LVAR_OK) return st;
  if (!rows_ok(q) || !o || !aligned(o, 16) || !M || !L || !lengths || !aligned(lengths, 4) || !aligned(counts, 4) || !aligned(M, 4) || !aligned(L, 4))
    return LVAR_EINVAL;
  if (!std::isfinite(scale) || scale <= 0.f || max_len < 0) return LVAR_EINVAL;
  const int64_t reach = (int64_t)cache.max_pages * cache.page_size;
  if (max_len > reach) max_len = (int)reach;
  // the stages of all tiles, counted in 31 bits on the device (a tile has at least 16 rows, a stage 128 keys)
  const int64_t rows = (int64_t)(H / cache.kv_heads) * Lq, tiles = (rows + 15) / 16 * cache.kv_heads * B;
  if (rows > kMostTokens || tiles > 0x7fffffffll / (max_len / 128 + 2)) return LVAR_EINVAL;
  p.q = (const bf16_t*)q.ptr; p.q_sb = q.stride_b; p.q_sh = q.stride_h; p.q_sr = q.stride_row;
  p.o = (bf16_t*)o; p.M = M; p.L = L;
  p.lengths = lengths; p.counts = counts;
  p.B = B; p.H = H; p.Lq = Lq; p.G = H / cache.kv_heads; p.causal = causal ? 1 : 0; p.max_len = max_len;
  p.c = scale * kLog2e;
  return launch_paged_attn(p, workspace, workspace_bytes, cache.head_dim, (hipStream_t)stream);
}

}  // extern "C"
