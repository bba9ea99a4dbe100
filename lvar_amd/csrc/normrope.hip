// Norms of queries and keys per head with the position rotation in the same pass, forward (into packed tensors, or with keys
// and values straight into a paged cache) and backward.
//
//   n = x * r,  r = 1 / max(|x|, eps)  or  1 / sqrt(mean(x^2) + eps)  or  1;     u = n * w;     y = R(pos) u
//   backward of g = dL/dy:  gu = R^T g,  dw = sum gu * n,  gn = gu * w,
//     dx = r (gn - n * sum(gn n) [/ d for the mean square]);  where |x| <= eps: dx = gn / eps
//
// Everything between the load and the store of a row is fp32; a result is rounded once.  A row is read by d / 8 lanes,
// 16 bytes each, its sums stay in registers.  A workgroup takes 256 / (d / 8) tokens and HC heads of them, so that the
// cosines and sines of a token (twice as many bytes as a row) are read once for HC rows.
#include "kvcache.h"

namespace lvar {

constexpr int NR_T = 256;
constexpr int64_t AXIS_TABLE_ROWS = 1 << 18;   // rows (tokens x heads) from which on a backward pass makes tables of its angles
typedef double f64x2 __attribute__((ext_vector_type(2)));

// Results of large forward launches go past the L2s, whoever reads them next mostly sits on another XCD: 2 x 16 x 4096 rows of q and of k
// 28.3 -> 26.4 us.  Gradients do so at every size (with a reader of each behind them, through the L2s / past them: 2 x 8 x 20 tokens 7.1 / 7.3 us,
// 2 x 16 x 256 9.7 / 9.3, 4096 58.3 / 60.6, 4 x 16 x 10521 342 / 340; the kernel alone over 10521 tokens 240 / 220).
template <bool STREAM>
__device__ __forceinline__ void put(bf16_t* to, u32x4 x) {
  if constexpr (STREAM) __builtin_nontemporal_store(x, (u32x4*)to);
  else *(u32x4*)to = x;
}

struct Angles {
  float c[8], s[8];   // pairs of the lane: 4 of them (interleaved) or 8 (halves)
  bool on;            // the lane's columns are among the rotated ones
  int partner;        // halves: lane (of the row) that holds the other halves of the pairs
  bool second;        // halves: this lane holds the second elements
};

// Sine and cosine of a number of turns in -1/2 .. 1/2, off by about a step of 32 bits: the nearest quarter turn is taken off in 64 bits, and what is
// left, at most pi / 4, goes into the power series of both up to x^9 and x^8 (their next terms are below 2^-28 and 2^-25 there).
__device__ __forceinline__ void sincos_of_turns(double t, float& s, float& c) {
  const float n = __builtin_rintf(4.f * (float)t);
  const float x = 6.28318530717958647692f * (float)__builtin_fma((double)n, -0.25, t), z = x * x;
  const float a = x * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
  const float b = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = (int)n & 3;   // (of NaN: 0, and a and b are NaN)
  const float u = q & 1 ? b : a, v = q & 1 ? a : b;
  s = q & 2 ? -u : u;
  c = (q + 1) & 2 ? -v : v;
}

// Sines and cosines of pairs pair .. pair + 3 of token i of sequence b.
__device__ __forceinline__ void four_angles(const NormRopeParams& p, int b, int i, int pair, float* s, float* c) {
  double turn[4] = {};
  for (int x = 0; x < p.axes; x++) {
    const int64_t at = b * p.pos_sb + x * p.pos_sa + i * p.pos_sl;
    const double pos = (p.pos64 == 2 ? (double)((const float*)p.positions)[at]
                        : p.pos64    ? (double)((const int64_t*)p.positions)[at]
                                     : (double)((const int32_t*)p.positions)[at]) * 0.15915494309189533577;   // 1 / (2 pi)
    const int64_t f = x * p.freq_sa + pair;
    if (p.freq32) {
      const f32x4 v = *(const f32x4*)((const float*)p.freqs + f);
#pragma unroll
      for (int e = 0; e < 4; e++) turn[e] = __builtin_fma(pos, (double)v[e], turn[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const f64x2 v = *(const f64x2*)((const double*)p.freqs + f + e);
        turn[e] = __builtin_fma(pos, v[0], turn[e]);
        turn[e + 1] = __builtin_fma(pos, v[1], turn[e + 1]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) sincos_of_turns(turn[e] - __builtin_rint(turn[e]), s[e], c[e]);
}

// Cosines and sines of the lane's pairs: of a row of the tables, or (AXES) of the sum over the axes of position times frequency, of token i of
// sequence b.  That sum is formed in 64 bits, as turns of which only the fraction is kept: a position of 2^20 times a frequency of 1 is known to
// 2^-4 of a radian in 32 bits.
template <int LPR, bool AXES>
__device__ __forceinline__ void load_angles(const NormRopeParams& p, int64_t row, int b, int i, int lane, Angles& a) {
  const int col = lane * 8, half = p.rot >> 1;
  a.on = (AXES || p.cos) && col < p.rot;
  a.second = false;
  a.partner = lane;
  int pair = col >> 1;
  if (!p.interleaved) {
    a.second = col >= half;
    pair = a.second ? col - half : col;
    a.partner = a.second ? lane - (half >> 3) : lane + (half >> 3);
  }
  if (!a.on) { a.partner = lane; return; }
  if constexpr (AXES) {
    // Four pairs per lane: those of two neighbouring columns are its own; of the halves, whose pairs two lanes share, each forms one half and they swap.
    if (!p.interleaved) pair += a.second ? 4 : 0;
    four_angles(p, b, i, pair, a.s, a.c);
    if (!p.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float so = __shfl(a.s[e], a.partner, LPR), co = __shfl(a.c[e], a.partner, LPR);
        a.s[4 + e] = a.second ? a.s[e] : so;
        a.c[4 + e] = a.second ? a.c[e] : co;
        a.s[e] = a.second ? so : a.s[e];
        a.c[e] = a.second ? co : a.c[e];
      }
    }
    return;
  }
  const float *cp = p.cos + row * p.cs_row + pair, *sp = p.sin + row * p.cs_row + pair;
  const f32x4 c0 = *(const f32x4*)cp, s0 = *(const f32x4*)sp;
#pragma unroll
  for (int e = 0; e < 4; e++) { a.c[e] = c0[e]; a.s[e] = s0[e]; }
  if (!p.interleaved) {
    const f32x4 c1 = *(const f32x4*)(cp + 4), s1 = *(const f32x4*)(sp + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) { a.c[4 + e] = c1[e]; a.s[4 + e] = s1[e]; }
  }
}

// f <- R f (BACK: R^T f).  Every lane takes part (the exchange of the halves).
template <int LPR, bool BACK, bool AXES>
__device__ __forceinline__ void rotate(const NormRopeParams& p, const Angles& a, float* f) {
  if (!AXES && !p.cos) return;
  if (p.interleaved) {
    if (!a.on) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = f[2 * e], y = f[2 * e + 1], s = BACK ? -a.s[e] : a.s[e];
      f[2 * e] = x * a.c[e] - y * s;
      f[2 * e + 1] = x * s + y * a.c[e];
    }
    return;
  }
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; e++) o[e] = __shfl(f[e], a.partner, LPR);
  if (!a.on) return;
  const float sign = a.second != BACK ? 1.f : -1.f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = f[e] * a.c[e] + sign * a.s[e] * o[e];
}

__device__ __forceinline__ void load_weight(const WeightView& w, int head, int lane, float* f) {
  if (w.mode == W_NONE) {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = 1.f;
  } else if (w.mode == W_HEAD) {
    const int64_t at = head * w.s_head;
    const float x = w.bf16 ? (float)((const bf16_t*)w.ptr)[at] : ((const float*)w.ptr)[at];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = x;
  } else {
    const int64_t at = head * w.s_head + lane * 8;
    if (w.bf16) {
      unpack8(*(const u32x4*)((const bf16_t*)w.ptr + at), f);
    } else {
      const f32x4 a = *(const f32x4*)((const float*)w.ptr + at), b = *(const f32x4*)((const float*)w.ptr + at + 4);
#pragma unroll
      for (int e = 0; e < 4; e++) { f[e] = a[e]; f[4 + e] = b[e]; }
    }
  }
}

// r of a row with this sum of squares; `flat`: |x| <= eps, where the l2 norm is a division by eps.  The reciprocal root is the
// hardware's (sums below its normal range scaled into it), off by up to one step of fp32, and one Newton step for the rest: with a root
// and a quotient rounded to nearest, a quarter of the instructions of a row went into these lines (append of 2 x 16 x 4096 tokens in e4m3
// 39.1 us, 37.7 with the step, 37.3 without it).  Of 6 x 16.8 M keys in e4m3, 95, 92 and 92 then have another code than in 64 bits.
template <int D>
__device__ __forceinline__ float norm_factor(const NormRopeParams& p, float ss, bool& flat) {
  flat = false;
  if (p.norm == NORM_NONE) return 1.f;
  if (p.norm == NORM_RMS) ss = ss * (1.f / D) + p.eps;
  const bool tiny = ss < 0x1p-100f;
  const float sc = tiny ? ss * 0x1p100f : ss;
  float r = __builtin_amdgcn_rsqf(sc);
  const float rest = __builtin_fmaf(-sc * r, r, 1.f);
  r = __builtin_fabsf(rest) < 0x1p-10f ? __builtin_fmaf(0.5f * r, rest, r) : r;   // (not of 0, infinity and NaN)
  r *= tiny ? 0x1p50f : 1.f;
  if (p.norm == NORM_L2 && ss * r <= p.eps) {   // ss * r = |x| (0 * inf, the norm of a zero row, is NaN)
    flat = true;
  }
  if (p.norm == NORM_L2 && ss == 0.f) flat = true;
  return flat ? p.inv_eps : r;
}

// t / L by a multiplication (see division_by): 31-bit t
__device__ __forceinline__ int sequence_of(const NormRopeParams& p, int t) {
  const uint32_t h = __umulhi(p.div_mul, (uint32_t)t);
  return (int)((h + (((uint32_t)t - h) >> p.div_s1)) >> p.div_s2);
}

__device__ __forceinline__ int64_t table_row(const NormRopeParams& p, int b, int i, int64_t base) {
  int64_t pos = base + i;
  if (p.positions) {
    const int64_t at = b * p.pos_sb + i * p.pos_sl;
    pos = p.pos64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
  }
  return pos < 0 ? 0 : pos >= p.table_rows ? p.table_rows - 1 : pos;
}

// chunks of HC heads: those of q (unless keys are written as they are), of k, and when appending of v
template <int HC>
__host__ __device__ __forceinline__ int chunks_of(const NormRopeParams& p, bool append) {
  const int nk = (p.Hkv + HC - 1) / HC;
  return (append && p.ready ? 0 : (p.H + HC - 1) / HC) + (append ? 2 * nk : nk);
}

// AXES: angles from several position axes, formed by the lanes that use them (10 operations of 64 bits per angle and axis, about 25 of 32 bits): 8 x 4096
// tokens of 32 + 8 heads of 128 with three axes 140 us, 4.8 TB/s; 2 x 16 heads of 4096 into an 8-bit cache 39.3 us, as by tables.
template <int D, int HC, bool APPEND, bool AXES = false>
__global__ __launch_bounds__(NR_T) void norm_rope_kernel(const NormRopeParams p) {
  constexpr int LPR = D / 8, RPB = NR_T / LPR;
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR;
  // heads fastest: the rows of a token lie next to each other in a fused projection (heads slowest, so that workgroups in flight
  // read 1 KiB pieces 12 KiB apart: 140 us where this takes 126, 4 x 10521 tokens of 32 heads)
  const int T = p.B * p.L, chunks_all = chunks_of<HC>(p, APPEND), t_own = (int)(blockIdx.x / chunks_all) * RPB + g;
  const bool live = t_own < T;
  const int t = live ? t_own : T - 1;
  const int b = sequence_of(p, t), i = t - b * p.L;
  // chunks of heads: those of q, then k, then v
  const int nq = APPEND && p.ready ? 0 : (p.H + HC - 1) / HC, nk = (p.Hkv + HC - 1) / HC;
  int c = blockIdx.x % chunks_all;
  const int which = c < nq ? 0 : c < nq + nk ? 1 : 2;
  c -= which == 0 ? 0 : which == 1 ? nq : nq + nk;
  const int heads = which == 0 ? p.H : p.Hkv, h0 = c * HC;
  const bf16_t* x = which == 0 ? p.q : which == 1 ? p.k : p.v;
  const int64_t sb = which == 0 ? p.q_sb : which == 1 ? p.k_sb : p.v_sb;
  const int64_t sh = which == 0 ? p.q_sh : which == 1 ? p.k_sh : p.v_sh;
  const int64_t sr = which == 0 ? p.q_sr : which == 1 ? p.k_sr : p.v_sr;
  const bf16_t* row = x + b * sb + i * sr + lane * 8;

  u32x4 in[HC];
#pragma unroll
  for (int j = 0; j < HC; j++) in[j] = *(const u32x4*)(row + (int64_t)min(h0 + j, heads - 1) * sh);

  const int64_t base = APPEND ? p.start[b] : 0;
  const bool plain = APPEND && (which == 2 || p.ready);   // written as it is
  Angles a;
  a.on = false;
  if (!plain && (AXES || p.cos)) load_angles<LPR, AXES>(p, AXES ? 0 : table_row(p, b, i, base), b, i, lane, a);
  // One factor for all columns commutes with the rotation and comes last: the rotation of bf16 values costs two roundings instead of three
  // or four (of 6 x 16.8 M keys in e4m3, 92 have another code than in 64 bits, 135 with the factor first).  Halved angles, so that the largest
  // values do not overflow.
  const float both = a.on ? 2.f : 1.f;
  if (a.on) {
#pragma unroll
    for (int e = 0; e < 8; e++) { a.c[e] *= 0.5f; a.s[e] *= 0.5f; }
  }

  bool place = false;
  int page = 0, slot = 0;
  if (APPEND && which != 0) place = live && (!p.counts || i < p.counts[b]) && find_row(p.cache, b, base + i, page, slot);

  const WeightView& w = which == 0 ? p.wq : p.wk;
#pragma unroll
  for (int j = 0; j < HC; j++) {
    const int head = h0 + j;
    if (head >= heads) break;
    float f[8];
    unpack8(in[j], f);
    if (!plain) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) ss += f[e] * f[e];
      ss = row_sum<LPR>(ss);
      bool flat;
      const float r = norm_factor<D>(p, ss, flat);
      float wf[8];
      load_weight(w, head, lane, wf);
      const bool columns = w.mode == W_COLUMN;
      const float last = (columns ? 1.f : r * wf[0]) * both;
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] *= columns ? r * wf[e] : 1.f;
      rotate<LPR, false, AXES>(p, a, f);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] *= last;
    }
    if (!APPEND || which == 0) {
      bf16_t* out = which == 0 ? p.oq : p.ok;
      if (live) put<(HC > 1)>(out + (((int64_t)b * heads + head) * p.L + i) * D + lane * 8, pack8u(f));
    } else {
      const int64_t at = page * p.cache.s_page + head * p.cache.s_head + slot * p.cache.s_row;
      uint8_t* pages = which == 1 ? p.cache.k : p.cache.v;
      if (p.cache.k_exp) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, finite_abs_bits(f[e]));
        const uint32_t byte = exp_byte(row_umax<LPR>(top));
        const u32x2 codes = codes8(f, byte);
        if (place) {
          *(u32x2*)(pages + at + lane * 8) = codes;
          if (lane == 0) (which == 1 ? p.cache.k_exp : p.cache.v_exp)[page * p.cache.e_page + head * p.cache.e_head + slot] = (uint8_t)byte;
        }
      } else if (place) {
        *(u32x4*)(pages + at + lane * 16) = plain ? in[j] : pack8u(f);
      }
    }
  }
}

// Constants of the division of 32-bit numbers by L (rounded-up reciprocal, Granlund and Montgomery 1994, figure 4.1).
static void division_by(NormRopeParams& p) {
  const uint32_t L = (uint32_t)p.L;
  int l = 0;
  while ((1ull << l) < L) l++;
  p.div_mul = (uint32_t)(((1ull << 32) * ((1ull << l) - L)) / L + 1);
  p.div_s1 = l < 1 ? l : 1;
  p.div_s2 = l - 1 > 0 ? l - 1 : 0;
}

template <int D, int HC>
static bool launch_fwd(const NormRopeParams& p, bool append, hipStream_t s) {
  constexpr int RPB = NR_T / (D / 8);
  const int64_t groups = (int64_t)chunks_of<HC>(p, append) * ((p.B * p.L + RPB - 1) / RPB);
  if (!grid_fits(groups, NR_T)) return false;
  if constexpr (D >= 64) {   // (head dimensions of a cache)
    if (append) {
      if (p.freqs) hipLaunchKernelGGL((norm_rope_kernel<D, HC, true, true>), dim3((uint32_t)groups), dim3(NR_T), 0, s, p);
      else hipLaunchKernelGGL((norm_rope_kernel<D, HC, true>), dim3((uint32_t)groups), dim3(NR_T), 0, s, p);
      return true;
    }
  }
  if (p.freqs) hipLaunchKernelGGL((norm_rope_kernel<D, HC, false, true>), dim3((uint32_t)groups), dim3(NR_T), 0, s, p);
  else hipLaunchKernelGGL((norm_rope_kernel<D, HC, false>), dim3((uint32_t)groups), dim3(NR_T), 0, s, p);
  return true;
}

template <int D>
static bool launch_fwd_d(const NormRopeParams& p, bool append, hipStream_t s) {
  // Four heads per workgroup once such workgroups are four per compute unit, one head before that (latency is the time there).
  constexpr int RPB = NR_T / (D / 8);
  const int64_t tiles = (int64_t)(p.B * p.L + RPB - 1) / RPB;
  return tiles * chunks_of<4>(p, append) >= 4ll * device_cus() ? launch_fwd<D, 4>(p, append, s) : launch_fwd<D, 1>(p, append, s);
}

int launch_norm_rope(NormRopeParams p, int head_dim, bool append, hipStream_t s) {
  division_by(p);
  p.inv_eps = 1.f / p.eps;
  bool ok = true;
  switch (head_dim) {
    case 16: if (append) return LVAR_EUNSUPPORTED; ok = launch_fwd_d<16>(p, append, s); break;
    case 32: if (append) return LVAR_EUNSUPPORTED; ok = launch_fwd_d<32>(p, append, s); break;
    case 64: ok = launch_fwd_d<64>(p, append, s); break;
    case 128: ok = launch_fwd_d<128>(p, append, s); break;
    case 256: ok = launch_fwd_d<256>(p, append, s); break;
    default: return LVAR_EUNSUPPORTED;
  }
  if (!ok) return LVAR_EINVAL;
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

// ---- backward ----

// Workgroup (blk, chunk): tokens blk * RPB + g, + nblk * RPB, ... of up to NB_HC heads of q or of k.  The weight gradients of its
// heads stay in registers over all its tokens and meet in LDS once, in a fixed order: row `blk` of the partial sums.
template <int D, bool DW, bool AXES>
__device__ __forceinline__ void norm_rope_bwd_item(const NormRopeParams& p, float* red) {
  constexpr int LPR = D / 8, RPB = NR_T / LPR, HC = NB_HC;
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR;
  const int T = p.B * p.L;
  const int nq = (p.H + HC - 1) / HC, nc = chunks_of<HC>(p, false);
  const int blk = blockIdx.x / nc, own = blockIdx.x % nc;
  const bool isq = own < nq;
  const int h0 = (isq ? own : own - nq) * HC;
  const int heads = isq ? p.H : p.Hkv;
  const bf16_t *x = isq ? p.q : p.k, *gy = isq ? p.gq : p.gk;
  bf16_t* dx = isq ? p.dq : p.dk;
  const int64_t sb = isq ? p.q_sb : p.k_sb, sh = isq ? p.q_sh : p.k_sh, sr = isq ? p.q_sr : p.k_sr;
  const int64_t db = isq ? p.dq_sb : p.dk_sb, dh = isq ? p.dq_sh : p.dk_sh, dr = isq ? p.dq_sr : p.dk_sr;
  const WeightView& w = isq ? p.wq : p.wk;
  float* part = isq ? p.pq : p.pk;
  void* done = isq ? p.dqw : p.dkw;

  float acc[DW ? HC : 1][8] = {};
  for (int t0 = blk * RPB; t0 < T; t0 += p.nblk * RPB) {
    const bool live = t0 + g < T;
    const int t = live ? t0 + g : T - 1;
    const int b = sequence_of(p, t), i = t - b * p.L;
    u32x4 xin[HC], gin[HC];
#pragma unroll
    for (int j = 0; j < HC; j++) {
      const int head = min(h0 + j, heads - 1);
      xin[j] = *(const u32x4*)(x + b * sb + head * sh + i * sr + lane * 8);
      gin[j] = *(const u32x4*)(gy + (((int64_t)b * heads + head) * p.L + i) * D + lane * 8);
    }
    Angles a;
    a.on = false;
    if (AXES || p.cos) load_angles<LPR, AXES>(p, AXES ? 0 : table_row(p, b, i, 0), b, i, lane, a);
#pragma unroll
    for (int j = 0; j < HC; j++) {
      const int head = h0 + j;
      if (head >= heads) break;
      float n[8], gu[8], wf[8];
      unpack8(xin[j], n);
      unpack8(gin[j], gu);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) ss += n[e] * n[e];
      ss = row_sum<LPR>(ss);
      bool flat;
      const float r = norm_factor<D>(p, ss, flat);
      rotate<LPR, true, AXES>(p, a, gu);
      load_weight(w, head, lane, wf);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        n[e] *= r;
        if constexpr (DW) { if (live) acc[j][e] += gu[e] * n[e]; }
        gu[e] *= wf[e];
        dot += gu[e] * n[e];
      }
      dot = row_sum<LPR>(dot);
      if (p.norm == NORM_RMS) dot *= 1.f / D;
      if (p.norm == NORM_NONE || flat) dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) gu[e] = r * (gu[e] - n[e] * dot);
      if (live) put<true>(dx + b * db + head * dh + i * dr + lane * 8, pack8u(gu));
    }
  }
  if constexpr (DW) {
    if (!part && !done) return;
    const bool shared = w.s_head == 0;   // one gradient for all heads: a partial row per workgroup, not per head
    if (shared) {
#pragma unroll
      for (int j = 1; j < HC; j++)       // (heads beyond the last one have added nothing)
#pragma unroll
        for (int e = 0; e < 8; e++) acc[0][e] += acc[j][e];
    }
    const int chunk = h0 / HC, chunks = (heads + HC - 1) / HC;
#pragma unroll
    for (int j = 0; j < HC; j++) {
      if (shared ? j > 0 : h0 + j >= heads) break;
#pragma unroll
      for (int e = 0; e < 8; e++) red[g * D + lane * 8 + e] = acc[j][e];
      __syncthreads();
      const int64_t at = shared ? (int64_t)blk * chunks + chunk : (int64_t)blk * heads + h0 + j;
      float sum = 0.f;
      if ((int)threadIdx.x < D)
        for (int r = 0; r < RPB; r++) sum += red[r * D + threadIdx.x];
      __syncthreads();
      if (!done) {
        if ((int)threadIdx.x < D) part[at * D + threadIdx.x] = sum;
        continue;
      }
      // the only row of its kind is the gradient
      int64_t to = shared ? 0 : h0 + j;
      if (w.mode == W_COLUMN) {
        to = to * D + threadIdx.x;
      } else {
        sum = row_sum<16>(sum);
        if (threadIdx.x % 16 == 0) red[threadIdx.x / 16] = sum;
        __syncthreads();
        sum = 0.f;
        for (int r = 0; r < D / 16; r++) sum += red[r];
        __syncthreads();
      }
      if ((int)threadIdx.x < (w.mode == W_COLUMN ? D : 1)) {
        if (w.bf16) ((bf16_t*)done)[to] = (bf16_t)sum;
        else ((float*)done)[to] = sum;
      }
    }
  }
}

template <int D, bool DW>
__global__ __launch_bounds__(NR_T) void norm_rope_bwd_kernel(const NormRopeParams p) {
  __shared__ float red[DW ? NR_T * 8 : 1];
  norm_rope_bwd_item<D, DW, false>(p, red);
}

template <int D, bool DW>
__global__ __launch_bounds__(NR_T) void norm_axes_bwd_kernel(const NormRopeParams p) {
  __shared__ float red[DW ? NR_T * 8 : 1];
  norm_rope_bwd_item<D, DW, true>(p, red);
}

// A workgroup per (head, 32 columns) of a gradient with columns, per head of one without; a gradient shared by the heads has one
// "head" whose rows are all partial rows.  Sums in a fixed order.
__global__ __launch_bounds__(1024) void weight_grad_kernel(const WeightGradParams w) {
  __shared__ float red[32][33];
  const int k = blockIdx.z;
  if (!w.out[k] || (int)blockIdx.x >= w.heads[k]) return;
  const bool scalar = w.cols[k] == 1;
  if (scalar ? blockIdx.y > 0 : (int)blockIdx.y * 32 >= w.D) return;
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const float* part = w.part[k] + (int64_t)blockIdx.x * w.D;
  const int64_t rs = (int64_t)w.heads[k] * w.D;
  float sum = 0.f;
  // (loads in runs of 8 whose end is clamped and not branched over: they are in flight together)
  if (scalar) {
    const int n = w.rows[k] * w.D, shift = 31 - __builtin_clz(w.D);
    for (int at = threadIdx.x; at < n; at += 8 * 1024) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int x = min(at + u * 1024, n - 1);
        v[u] = part[(x >> shift) * rs + (x & (w.D - 1))];
      }
#pragma unroll
      for (int u = 0; u < 8; u++) sum += at + u * 1024 < n ? v[u] : 0.f;
    }
  } else {
    const int col = blockIdx.y * 32 + cl;
    for (int r = rl; r < w.rows[k]; r += 8 * 32) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = part[min(r + u * 32, w.rows[k] - 1) * rs + min(col, w.D - 1)];
#pragma unroll
      for (int u = 0; u < 8; u++) sum += r + u * 32 < w.rows[k] ? v[u] : 0.f;
    }
  }
  red[rl][cl] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 32; r++) s += red[r][cl];
    int64_t at = (int64_t)blockIdx.x * w.D + blockIdx.y * 32 + cl;
    bool mine = (int)blockIdx.y * 32 + cl < w.D;
    if (scalar) {
      s = row_sum<32>(s);
      at = blockIdx.x;
      mine = cl == 0;
    }
    if (mine) {
      if (w.bf16[k]) ((bf16_t*)w.out[k])[at] = (bf16_t)s;
      else ((float*)w.out[k])[at] = s;
    }
  }
}

// ---- tables of the angles of a call ----

// A large backward pass reads cosines and sines from tables that a launch ahead of it writes to scratch memory, with the row of every token where sequences differ: the
// angles are formed once, not once per pair of heads.  Formed in place / from tables, both launches, 32 + 8 heads of 128 with three axes, pairs of
// neighbours: 410 tokens 12.2 / 14.7 us, 3280 34.5 / 36.0, 8192 65.5 / 64.2, 32768 285 / 266; of halves 12.3 / 14.9, 35.3 / 35.3, 68.1 / 65.0, 308 / 277.
// The forward launches, whose workgroups form them for four heads and do not loop, gain nothing (2 x 32 heads of 4096 into a cache 39.7 / 41.1).
__global__ __launch_bounds__(NR_T) void axis_tables_kernel(const NormRopeParams p, float* cos, float* sin, int32_t* row_of, int rows) {
  const int quads = p.rot >> 3;                                  // of pairs
  const int64_t at = (int64_t)blockIdx.x * NR_T + threadIdx.x;
  const int64_t r = at / quads;
  if (row_of && at < rows) row_of[at] = (int)at;
  if (r >= rows) return;
  const int q = (int)(at - r * quads), b = (int)(r / p.L), i = (int)(r - (int64_t)b * p.L);
  float s[4], c[4];
  four_angles(p, b, i, 4 * q, s, c);
  *(f32x4*)(cos + r * (p.rot >> 1) + 4 * q) = f32x4{c[0], c[1], c[2], c[3]};
  *(f32x4*)(sin + r * (p.rot >> 1) + 4 * q) = f32x4{s[0], s[1], s[2], s[3]};
}

static int64_t axis_rows(const NormRopeParams& p) { return p.pos_sb ? (int64_t)p.B * p.L : p.L; }

int64_t axis_table_bytes(const NormRopeParams& p) {
  if ((int64_t)p.B * p.L * (p.H + p.Hkv) < AXIS_TABLE_ROWS) return 0;
  return axis_rows(p) * p.rot * 4 + (p.pos_sb ? (int64_t)p.B * p.L * 4 : 0);
}

// Writes the tables and turns p into a call that reads them.
int launch_axis_tables(NormRopeParams& p, void* scratch, hipStream_t s) {
  const int64_t rows = axis_rows(p), half = p.rot >> 1;
  float *cos = (float*)scratch, *sin = cos + rows * half;
  int32_t* row_of = p.pos_sb ? (int32_t*)(sin + rows * half) : nullptr;   // (without, a token's row is its number: 250 us instead of 262 for the largest call above)
  const int64_t groups = (rows * (half >> 2) + NR_T - 1) / NR_T;
  if (!grid_fits(groups, NR_T)) return LVAR_EINVAL;
  hipLaunchKernelGGL(axis_tables_kernel, dim3((uint32_t)groups), dim3(NR_T), 0, s, p, cos, sin, row_of, (int)rows);
  p.cos = cos; p.sin = sin; p.cs_row = half; p.table_rows = (int)rows;
  p.positions = row_of; p.pos64 = 0; p.pos_sb = p.L; p.pos_sl = 1;
  p.freqs = nullptr;
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

// Rows of partial weight gradients: as many workgroups along the tokens as give every compute unit about eight, but no more than there are tiles.
// With `alone` (all weight gradients that are wanted are gradients per head), one for up to 8 tiles: its row is the gradient, without a second
// launch, in a kernel that stays shorter than its call (training passes of 2 x 8 heads of 20 tokens and of 8 x 16 heads of 16, bound by
// their host threads: 44.5 -> 40.7 us).
int norm_rope_bwd_blocks(int B, int H, int Hkv, int L, int head_dim, bool alone) {
  const int rpb = NR_T / (head_dim / 8), chunks = (H + NB_HC - 1) / NB_HC + (Hkv + NB_HC - 1) / NB_HC;
  const int64_t tiles = ((int64_t)B * L + rpb - 1) / rpb, want = (8ll * device_cus() + chunks - 1) / chunks;
  if (alone && tiles <= 8) return 1;
  return (int)(tiles < want ? tiles : want);
}

template <int D>
static void launch_bwd(const NormRopeParams& p, hipStream_t s) {
  const dim3 grid((uint32_t)chunks_of<NB_HC>(p, false) * (uint32_t)p.nblk);
  const bool weights = p.pq || p.pk || p.dqw || p.dkw;
  if (p.freqs) {
    if (weights) hipLaunchKernelGGL((norm_axes_bwd_kernel<D, true>), grid, dim3(NR_T), 0, s, p);
    else hipLaunchKernelGGL((norm_axes_bwd_kernel<D, false>), grid, dim3(NR_T), 0, s, p);
  } else if (weights) {
    hipLaunchKernelGGL((norm_rope_bwd_kernel<D, true>), grid, dim3(NR_T), 0, s, p);
  } else {
    hipLaunchKernelGGL((norm_rope_bwd_kernel<D, false>), grid, dim3(NR_T), 0, s, p);
  }
}

int launch_norm_rope_bwd(NormRopeParams p, int head_dim, hipStream_t s) {
  division_by(p);
  p.inv_eps = 1.f / p.eps;
  switch (head_dim) {
    case 16: launch_bwd<16>(p, s); break;
    case 32: launch_bwd<32>(p, s); break;
    case 64: launch_bwd<64>(p, s); break;
    case 128: launch_bwd<128>(p, s); break;
    case 256: launch_bwd<256>(p, s); break;
    default: return LVAR_EUNSUPPORTED;
  }
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

int launch_weight_grad(const WeightGradParams& w, hipStream_t s) {
  const int heads = w.heads[0] > w.heads[1] ? w.heads[0] : w.heads[1];
  hipLaunchKernelGGL(weight_grad_kernel, dim3(heads, (w.D + 31) / 32, 2), dim3(1024), 0, s, w);
  return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH;
}

}  // namespace lvar
