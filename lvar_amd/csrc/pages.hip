// The life of the pages of a cache: dropping, opening and forking the pages that a table names, with a count of names per page, and copying chosen
// tokens of a sequence to other pages.  Nothing of it comes from the host: a step captured in a graph is replayed with other lengths.
//
// All of it is latency: 192 samples of 48 prompts (240 rows, 1500 pages) drop 2.8, search 3.9, fork 7.5 (50 MB read and written), open 5.6 us; 4 samples of
// one 2.5 + 3.4 + 3.4 + 2.9.
//
// Which free page (refs <= 0) a call hands out is fixed: the lowest ones, in the order of rows and entries.  One workgroup finds them: it adds up
// what the rows want, scans the counts until it has as many, and deals them out.  Counts change by integer additions, whose order does not matter.
#include "kvcache.h"

namespace lvar {

// threads of the search; pages that it keeps in LDS; rows of a table of which pairs are checked
constexpr int PG_FEW = 64, PG_SOME = 256, PG_T = 1024, PG_LIST = 4096, PG_MARKS = 65536 / 32;

// Sum over the workgroup ahead of this thread, and of all; `part` has a place for every wave.
template <int T, class I>
__device__ __forceinline__ I prefix(I x, I* part, I& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  I sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const I up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  if constexpr (T == 64) {
    total = __shfl(sum, 63, 64);
    return sum - x;
  }
  __syncthreads();   // (part may still be read from the call before)
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 64; w++) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + sum - x;
}

// Which of four pages from g on are free, a bit each
__device__ __forceinline__ int free_of(const PagesParams& p, int g) {
  int bits = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) bits |= (g + e < p.num_pages && p.refs[min(g + e, p.num_pages - 1)] <= 0 ? 1 : 0) << e;
  return bits;
}

// The first N free pages into `list`; how many there are.  `bits`: free_of() this thread's first pages, asked for ahead of what N needs.
template <int T>
__device__ __forceinline__ int find_free(const PagesParams& p, int bits, int N, int* list, int* part) {
  int found = 0;
  for (int g0 = 0; g0 < p.num_pages && found < N; g0 += 4 * T) {
    const int g = g0 + 4 * (int)threadIdx.x;
    if (g0 > 0) bits = free_of(p, g);
    int all, at = found + prefix<T>(__builtin_popcount(bits), part, all);
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (bits >> e & 1) {
        if (at < N) list[at] = g + e;
        at++;
      }
    found = min(found + all, N);
  }
  __syncthreads();
  return found;
}

template <int T>
__global__ __launch_bounds__(T) void pages_alloc_kernel(const PagesParams p) {
  __shared__ int64_t part64[T / 64];
  __shared__ int part[T / 64], lds_list[PG_LIST], want_at[T], want_n[T], want_base[T];
  const int tid = threadIdx.x, bits = free_of(p, 4 * tid);
  int N = 0, at = 0, n = 0, before = 0;
  // entries that row r0 + tid wants, and how many the rows ahead of it do (no more than there are pages)
  auto wants = [&](int r0, int done) {
    const int r = r0 + tid;
    at = n = 0;
    if (r < p.n) {
      at = max(0, min(p.first[r], p.max_pages));
      n = max(0, max(0, min(p.last[r], p.max_pages)) - at);
    }
    int64_t all;
    const int64_t x = prefix<T>((int64_t)n, part64, all);
    before = (int)min(done + x, (int64_t)p.num_pages);
    return (int)min(done + all, (int64_t)p.num_pages);
  };
  for (int r0 = 0; r0 < p.n; r0 += T) N = wants(r0, N);
  int* list = N <= PG_LIST ? lds_list : p.scratch;
  const int found = find_free<T>(p, bits, N, list, part);
  // lanes of a row: as many as there are threads for, 8 at least
  const int lanes = 31 - __builtin_clz(max(8, T / max(1, min(p.n, T))));
  int done = 0;
  for (int r0 = 0; r0 < p.n; r0 += T) {
    if (p.n > T) done = wants(r0, done);
    __syncthreads();
    want_at[tid] = at;
    want_n[tid] = n;
    want_base[tid] = before;
    __syncthreads();
    const int rows = min(T, p.n - r0);
    for (int r = tid >> lanes; r < rows; r += T >> lanes) {
      int* to = p.table + (r0 + r) * p.table_stride + want_at[r];
      const int64_t base = want_base[r];
      for (int e = tid & ((1 << lanes) - 1); e < want_n[r]; e += 1 << lanes) {
        const int page = base + e < found ? list[base + e] : -1;
        to[e] = page;
        if (page >= 0) p.refs[page] = 1;
      }
    }
  }
}

// What becomes of fork r, from pages_fork_find_kernel to pages_fork_kernel: the page for the started one, or one of these.
constexpr int FORK_NOTHING = -1, FORK_LEFT_OUT = -2;

// Pairs that would make the result depend on an order are left out: two with the same target, and a target that is the source of another.
template <int T>
__global__ __launch_bounds__(T) void pages_fork_find_kernel(const PagesParams p) {
  __shared__ int part[T / 64], lds_list[PG_LIST];
  __shared__ uint32_t sources[PG_MARKS], once[PG_MARKS], twice[PG_MARKS];   // a bit per row of the table
  const int tid = threadIdx.x, bits = free_of(p, 4 * tid);
  int s = -1, t = -1;
  auto pair = [&](int r) {
    s = r < p.n ? p.source[r] : -1;
    t = r < p.n ? p.target[r] : -1;
    return s >= 0 && s < p.rows && t >= 0 && t < p.rows && s != t;
  };
  for (int i = tid; i < (p.rows + 31) / 32; i += T) sources[i] = once[i] = twice[i] = 0;
  __syncthreads();
  bool ok = false;
  for (int r0 = 0; r0 < p.n; r0 += T) {
    ok = pair(r0 + tid);
    if (!ok) continue;
    atomicOr(sources + (s >> 5), 1u << (s & 31));
    if (atomicOr(once + (t >> 5), 1u << (t & 31)) >> (t & 31) & 1) atomicOr(twice + (t >> 5), 1u << (t & 31));
  }
  __syncthreads();
  int N = 0, before = 0, n = 0, state = 0;
  auto wants = [&](int r0, int done) {
    if (p.n > T) ok = pair(r0 + tid);
    state = FORK_LEFT_OUT;
    n = 0;
    if (ok && !((sources[t >> 5] | twice[t >> 5]) >> (t & 31) & 1)) {
      const int len = max(0, p.lengths[s]), whole = len >> p.shift;
      state = FORK_NOTHING;
      if (whole < p.max_pages && (len & ((1 << p.shift) - 1)) != 0) {
        const int page = p.table[s * p.table_stride + whole];
        n = page >= 0 && page < p.num_pages ? 1 : 0;
      }
    }
    int all;
    before = done + prefix<T>(n, part, all);
    return done + all;
  };
  for (int r0 = 0; r0 < p.n; r0 += T) N = wants(r0, N);
  N = min(N, p.num_pages);   // (a list that LDS does not hold is then of a pool that has its place behind the forks, see pages_scratch_ints)
  int* list = N <= PG_LIST ? lds_list : p.scratch + p.n;
  const int found = N > 0 ? find_free<T>(p, bits, N, list, part) : 0;
  int done = 0;
  for (int r0 = 0; r0 < p.n; r0 += T) {
    if (p.n > T) done = wants(r0, done);
    if (r0 + tid >= p.n) continue;
    if (n && before < found) {
      state = list[before];
      p.refs[state] = 1;
    }
    p.scratch[r0 + tid] = state;
  }
}

// Entries from keep[b] on name no page any more.
__global__ __launch_bounds__(256) void pages_free_kernel(const PagesParams p) {
  const int b = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x;
  if (e >= p.max_pages || (p.first && e < p.first[b])) return;
  int* at = p.table + b * p.table_stride + e;
  const int page = *at;
  if (page >= 0 && page < p.num_pages) atomicSub(p.refs + page, 1);
  if (page != -1) *at = -1;
}

// Fork r: the first workgroup of the row shares the whole pages and writes the rest of the target's row; all of them copy the rows of the started
// page, a head each.
__global__ __launch_bounds__(256) void pages_fork_kernel(const PagesParams p, const PagedView c, const int chunks) {
  const int r = blockIdx.y, head = blockIdx.x, tid = threadIdx.x, fresh = p.scratch[r];
  if (fresh == FORK_LEFT_OUT) return;
  const int s = p.source[r], t = p.target[r];
  const int len = max(0, p.lengths[s]), whole = min(len >> p.shift, p.max_pages);
  const int *from = p.table + s * p.table_stride;
  int* to = p.table + t * p.table_stride;
  const int old = fresh >= 0 ? from[whole] : -1;
  if (head == 0) {
    for (int e = tid; e < p.max_pages; e += 256) {
      const int page = e < whole ? from[e] : e == whole ? fresh : -1;
      to[e] = page;
      if (e < whole && page >= 0 && page < p.num_pages) atomicAdd(p.refs + page, 1);
    }
  }
  if (fresh < 0) return;
  const int rest = len & ((1 << p.shift) - 1);
  const int64_t a = old * c.s_page + head * c.s_head, z = fresh * c.s_page + head * c.s_head;
  const int per = 31 - __builtin_clz(chunks);
  for (int i = tid; i < rest << per; i += 256) {
    const int64_t at = (int64_t)(i >> per) * c.s_row + (i & (chunks - 1)) * 16;
    const u32x4 x = *(const u32x4*)(c.k + a + at), y = *(const u32x4*)(c.v + a + at);
    *(u32x4*)(c.k + z + at) = x;
    *(u32x4*)(c.v + z + at) = y;
  }
  if (c.k_exp) {
    const int64_t ea = old * c.e_page + head * c.e_head, ez = fresh * c.e_page + head * c.e_head;
    for (int i = tid; i < rest; i += 256) {
      c.k_exp[ez + i] = c.k_exp[ea + i];
      c.v_exp[ez + i] = c.v_exp[ea + i];
    }
  }
}

// Token i of a head in the pages of `out`: token keep[b, head, i] of `c`, as its bytes are.  A row is read by `1 << per` lanes, 16 bytes each of
// key and value.  Bound by memory, and by its round trips (table and position, then the row) where it is small: 2 x 16 heads keep 1052 of 10521 tokens of
// 128 in bf16 6.4 to 7.2 us, 4.8 to 5.4 TB/s read and written; 8 x 8 heads up to 4001 of 8191 in e4m3 15.5 us, 4.6 TB/s of rows of 128 bytes and their exponents.
__global__ __launch_bounds__(256) void pages_compact_kernel(const CompactParams p, const int per) {
  const int lane = threadIdx.x & ((1 << per) - 1), i = (blockIdx.x << (8 - per)) + (threadIdx.x >> per);
  const int head = blockIdx.y, b = blockIdx.z;
  if (i >= p.n || (p.counts && i >= p.counts[b])) return;
  const int64_t k = b * p.keep_sb + head * p.keep_sh + i * p.keep_si;
  const int64_t pos = p.keep64 ? ((const int64_t*)p.keep)[k] : (int64_t)((const int32_t*)p.keep)[k];
  int page, slot, to, to_slot;
  if (!find_row(p.out, b, i, to, to_slot)) return;
  const bool there = find_row(p.cache, b, pos, page, slot);
  const PagedView& c = p.cache;
  u32x4 x{}, y{};
  const int64_t at = page * c.s_page + head * c.s_head + slot * c.s_row + lane * 16;
  if (there) {
    x = *(const u32x4*)(c.k + at);
    y = *(const u32x4*)(c.v + at);
  }
  const int64_t z = to * c.s_page + head * c.s_head + to_slot * c.s_row + lane * 16;
  *(u32x4*)(c.k + z) = x;
  *(u32x4*)(c.v + z) = y;
  if (c.k_exp && lane == 0) {
    const int64_t ea = page * c.e_page + head * c.e_head + slot, ez = to * c.e_page + head * c.e_head + to_slot;
    c.k_exp[ez] = there ? c.k_exp[ea] : (uint8_t)127;
    c.v_exp[ez] = there ? c.v_exp[ea] : (uint8_t)127;
  }
}

static int status() { return hipGetLastError() == hipSuccess ? LVAR_OK : LVAR_ELAUNCH; }

// ints of scratch: what becomes of each fork, and pages that do not fit the LDS of the search
int64_t pages_scratch_ints(int forks, int num_pages) {
  return forks + (num_pages > PG_LIST ? num_pages : 0);
}

// Threads of a search.  One wave where it sees all pages at once and needs no barrier (33 pages: the search of four forks 4.8 -> 3.4 us, of four rows 5.3
// -> 2.9 us); four where they see them in two looks and hold all rows, 16 beyond (4 / 16 waves: 20 rows or forks on 1000 pages 3.4 / 5.1 and 3.6 / 4.6 us, 192 on 1500
// pages, all taken but the last 5.7 / 5.4 and 5.1 / 5.1, on 4096 7.8 / 6.0 and 6.9 / 5.8).
static int threads(const PagesParams& p) {
  return p.n <= PG_FEW && p.num_pages <= 4 * PG_FEW ? PG_FEW : p.n <= PG_SOME && p.num_pages <= 8 * PG_SOME ? PG_SOME : PG_T;
}

int launch_pages_alloc(const PagesParams& p, hipStream_t s) {
  const int t = threads(p);
  if (t == PG_FEW) hipLaunchKernelGGL(pages_alloc_kernel<PG_FEW>, dim3(1), dim3(PG_FEW), 0, s, p);
  else if (t == PG_SOME) hipLaunchKernelGGL(pages_alloc_kernel<PG_SOME>, dim3(1), dim3(PG_SOME), 0, s, p);
  else hipLaunchKernelGGL(pages_alloc_kernel<PG_T>, dim3(1), dim3(PG_T), 0, s, p);
  return status();
}

int launch_pages_free(const PagesParams& p, hipStream_t s) {
  hipLaunchKernelGGL(pages_free_kernel, dim3((p.max_pages + 255) / 256, p.rows), dim3(256), 0, s, p);
  return status();
}

int launch_pages_fork(const PagesParams& p, const PagedView& c, int row_bytes, hipStream_t s) {
  const int t = threads(p);
  if (t == PG_FEW) hipLaunchKernelGGL(pages_fork_find_kernel<PG_FEW>, dim3(1), dim3(PG_FEW), 0, s, p);
  else if (t == PG_SOME) hipLaunchKernelGGL(pages_fork_find_kernel<PG_SOME>, dim3(1), dim3(PG_SOME), 0, s, p);
  else hipLaunchKernelGGL(pages_fork_find_kernel<PG_T>, dim3(1), dim3(PG_T), 0, s, p);
  const int st = status();
  if (st != LVAR_OK) return st;
  hipLaunchKernelGGL(pages_fork_kernel, dim3(c.kv_heads, p.n), dim3(256), 0, s, p, c, row_bytes / 16);
  return status();
}

int launch_pages_compact(const CompactParams& p, int B, int row_bytes, hipStream_t s) {
  const int per = __builtin_ctz((unsigned)row_bytes / 16), rows = 256 >> per;
  const dim3 grid((p.n + rows - 1) / rows, p.cache.kv_heads, B);
  if (!grid_fits(grid.x, 256)) return LVAR_EINVAL;
  hipLaunchKernelGGL(pages_compact_kernel, grid, dim3(256), 0, s, p, per);
  return status();
}

}  // namespace lvar
