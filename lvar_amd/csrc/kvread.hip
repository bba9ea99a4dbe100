// Reading the paged cache back: token start[b] + i of sequence b into row i of packed bf16 keys and values, zeros behind the
// length (and where the table names no page), for the operators that take [B,H,L,d].  A copy: one or two bytes read and two
// written per element, bandwidth-bound.
#include "kvcache.h"

namespace lvar {

constexpr int KR_T = 256;

template <int D, bool F8>
__global__ __launch_bounds__(KR_T) void kv_read_kernel(const KvReadParams p) {
  constexpr int LPR = D / 8, RPB = KR_T / LPR;   // lanes per row, rows per workgroup
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int head = blockIdx.y, b = blockIdx.z;
  const int i = blockIdx.x * RPB + g;
  if (i >= p.Lmax) return;
  const int64_t pos = (int64_t)(p.start ? p.start[b] : 0) + i;
  int page, slot;
  const bool there = pos < p.lengths[b] && find_row(p.cache, b, pos, page, slot);
  u32x4 x[2] = {};
  if (there) {
    const int64_t at = page * p.cache.s_page + head * p.cache.s_head + slot * p.cache.s_row;
    if constexpr (F8) {
      const int64_t ea = page * p.cache.e_page + head * p.cache.e_head + slot;
      const u32x2 ck = *(const u32x2*)(p.cache.k + at + lane * 8), cv = *(const u32x2*)(p.cache.v + at + lane * 8);
      const float ek = exp_value(p.cache.k_exp[ea]), ev = exp_value(p.cache.v_exp[ea]);
      x[0] = values8(ck, ek);
      x[1] = values8(cv, ev);
    } else {
      x[0] = *(const u32x4*)(p.cache.k + at + lane * 16);
      x[1] = *(const u32x4*)(p.cache.v + at + lane * 16);
    }
  }
  const int64_t out = (((int64_t)b * p.cache.kv_heads + head) * p.Lmax + i) * D + lane * 8;
  *(u32x4*)(p.k + out) = x[0];
  *(u32x4*)(p.v + out) = x[1];
}

template <int D>
static int launch_d(const KvReadParams& p, hipStream_t s) {
  constexpr int RPB = KR_T / (D / 8);
  const dim3 grid((p.Lmax + RPB - 1) / RPB, p.cache.kv_heads, p.B);
  if (!grid_fits(grid.x, KR_T)) return LVAR_EINVAL;
  if (p.cache.k_exp) hipLaunchKernelGGL((kv_read_kernel<D, true>), grid, dim3(KR_T), 0, s, p);
  else hipLaunchKernelGGL((kv_read_kernel<D, false>), grid, dim3(KR_T), 0, s, p);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

int launch_kv_read(const KvReadParams& p, int head_dim, hipStream_t s) {
  if (head_dim == 128) return launch_d<128>(p, s);
  if (head_dim == 64) return launch_d<64>(p, s);
  if (head_dim == 256) return launch_d<256>(p, s);
  return LVAR_EUNSUPPORTED;
}

}  // namespace lvar
