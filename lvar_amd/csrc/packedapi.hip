// extern "C" entry points of the attention over packed sequences: argument checks and parameter packing.
#include <cmath>
#include "packed.h"

using namespace lvar;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// rows that the kernels read (with 31 bits of byte offsets, and 32 for tiles that end behind them, which reach less than 512 rows further) or write
bool rows_ok(const lvar_tensor_t& t, int tokens, int head_dim) {
  if (tokens == 0) return true;
  return t.ptr && aligned(t.ptr, 16) && t.stride_h % 8 == 0 && t.stride_row % 8 == 0 && t.stride_row >= 0 &&
         (tokens == 1 || t.stride_row <= (1 << 20)) && (int64_t)(tokens - 1) * t.stride_row * 2 + 2 * head_dim < 0x7fffffffll;
}

bool sizes_ok(int batch, int tokens, int k_tokens, int H, int kv_heads) {
  return batch > 0 && batch <= (1 << 24) && tokens >= 0 && k_tokens >= 0 && kv_heads > 0 && H > 0 && H % kv_heads == 0 && H <= 16384;
}

int fill(PackedParams& p, const lvar_tensor_t& q, const lvar_tensor_t& k, const lvar_tensor_t& v, const lvar_tensor_t& o, const int32_t* offsets,
         const int32_t* k_offsets, float* M, float* L, int batch, int tokens, int k_tokens, int H, int kv_heads, int head_dim, int causal, float scale) {
  if (!sizes_ok(batch, tokens, k_tokens, H, kv_heads)) return LVAR_EINVAL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LVAR_EUNSUPPORTED;
  if (!offsets || !k_offsets || !aligned(offsets, 4) || !aligned(k_offsets, 4) || !std::isfinite(scale) || scale <= 0.f) return LVAR_EINVAL;
  // c and its reciprocal are used
  if (!std::isnormal(scale * kLog2e) || !std::isfinite(1.f / (scale * kLog2e))) return LVAR_EINVAL;
  if (!rows_ok(q, tokens, head_dim) || !rows_ok(o, tokens, head_dim) || !rows_ok(k, k_tokens, head_dim) || !rows_ok(v, k_tokens, head_dim)) return LVAR_EINVAL;
  if (tokens > 0 && (!M || !L || !aligned(M, 4) || !aligned(L, 4))) return LVAR_EINVAL;
  p.q = (const bf16_t*)q.ptr; p.q_sh = q.stride_h; p.q_sr = q.stride_row;
  p.k = (const bf16_t*)k.ptr; p.k_sh = k.stride_h; p.k_sr = k.stride_row;
  p.v = (const bf16_t*)v.ptr; p.v_sh = v.stride_h; p.v_sr = v.stride_row;
  p.o = (bf16_t*)o.ptr; p.o_sh = o.stride_h; p.o_sr = o.stride_row;
  p.M = M; p.L = L; p.q_off = offsets; p.k_off = k_offsets;
  p.B = batch; p.T = tokens; p.Tk = k_tokens; p.H = H; p.Hkv = kv_heads; p.G = H / kv_heads; p.causal = causal ? 1 : 0;
  p.scale = scale; p.c = scale * kLog2e;
  return LVAR_OK;
}

}  // namespace

extern "C" {

int64_t lvar_packed_attn_fwd_workspace_bytes(int batch, int tokens, int k_tokens, int H, int kv_heads, int head_dim, int causal) {
  if (!sizes_ok(batch, tokens, k_tokens, H, kv_heads)) return LVAR_EINVAL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LVAR_EUNSUPPORTED;
  PackedParams p{};
  p.B = batch; p.T = tokens; p.Tk = k_tokens; p.H = H; p.Hkv = kv_heads; p.G = H / kv_heads; p.causal = causal ? 1 : 0;
  return packed_fwd_bytes(p, head_dim);
}

int lvar_packed_attn_fwd(lvar_tensor_t q, lvar_tensor_t k, lvar_tensor_t v, lvar_tensor_t o, const int32_t* offsets, const int32_t* k_offsets, float* M,
                         float* L, void* workspace, int64_t workspace_bytes, int batch, int tokens, int k_tokens, int H, int kv_heads, int head_dim, int causal, float scale, void* stream) {
  PackedParams p{};
  const int st = fill(p, q, k, v, o, offsets, k_offsets, M, L, batch, tokens, k_tokens, H, kv_heads, head_dim, causal, scale);
  if (st != LVAR_OK || tokens == 0) return st;
  const int64_t bytes = packed_fwd_bytes(p, head_dim);
  if (bytes > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < bytes)) return LVAR_EINVAL;
  return launch_packed_fwd(p, workspace, head_dim, (hipStream_t)stream);
}

int64_t lvar_packed_attn_bwd_workspace_bytes(int batch, int tokens, int k_tokens, int H, int kv_heads, int head_dim, int causal) {
  if (!sizes_ok(batch, tokens, k_tokens, H, kv_heads)) return LVAR_EINVAL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return LVAR_EUNSUPPORTED;
  PackedParams p{};
  p.B = batch; p.T = tokens; p.Tk = k_tokens; p.H = H; p.Hkv = kv_heads; p.G = H / kv_heads; p.causal = causal ? 1 : 0;
  return packed_bwd_bytes(p, head_dim);
}

int lvar_packed_attn_bwd(lvar_tensor_t q, lvar_tensor_t k, lvar_tensor_t v, lvar_tensor_t o, lvar_tensor_t go, const int32_t* offsets,
                         const int32_t* k_offsets, const float* M, const float* L, lvar_tensor_t dq, lvar_tensor_t dk, lvar_tensor_t dv, void* workspace,
                         int64_t workspace_bytes, int batch, int tokens, int k_tokens, int H, int kv_heads, int head_dim, int causal, float scale,
                         void* stream) {
  PackedParams p{};
  const int st = fill(p, q, k, v, o, offsets, k_offsets, (float*)M, (float*)L, batch, tokens, k_tokens, H, kv_heads, head_dim, causal, scale);
  if (st != LVAR_OK) return st;
  if (!rows_ok(go, tokens, head_dim) || (dq.ptr && !rows_ok(dq, tokens, head_dim)) || (dk.ptr && !rows_ok(dk, k_tokens, head_dim)) ||
      (dv.ptr && !rows_ok(dv, k_tokens, head_dim)))
    return LVAR_EINVAL;
  const int64_t bytes = packed_bwd_bytes(p, head_dim);
  if (bytes > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < bytes)) return LVAR_EINVAL;
  p.g = (const bf16_t*)go.ptr; p.g_sh = go.stride_h; p.g_sr = go.stride_row;
  p.dq = (bf16_t*)dq.ptr; p.dq_sh = dq.stride_h; p.dq_sr = dq.stride_row;
  p.dk = (bf16_t*)dk.ptr; p.dk_sh = dk.stride_h; p.dk_sr = dk.stride_row;
  p.dv = (bf16_t*)dv.ptr; p.dv_sh = dv.stride_h; p.dv_sr = dv.stride_row;
  return launch_packed_bwd(p, workspace, head_dim, (hipStream_t)stream);
}

}  // extern "C"
