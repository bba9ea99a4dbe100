// The life of the pages of a cache: dropping, opening and forking the pages that a table names, with a count of names per page, and copying chosen
// tokens of a sequence to other pages.  Nothing of it comes from the host: a step captured in a graph is replayed with other lengths.
//
// Which free page (refs <= 0) a call hands out is fixed: the lowest ones, in the order of rows and entries.  One workgroup finds them: it adds up
// what the rows want, scans the counts until it has as many, and deals them out.  Counts change by integer additions, whose order does not matter.
#include "kvcache.h"

namespace lvar {

constexpr int PG_T = 1024, PG_LIST = 8192, PG_ROWS = 4096;   // threads; pages and rows that the search keeps in LDS

// Sum over the workgroup ahead of this thread, and of all; `part` has a place for every wave.
template <class I>
__device__ __forceinline__ I prefix(I x, I* part, I& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  I sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const I up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  __syncthreads();   // (part may still be read from the call before)
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PG_T / 64; w++) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + sum - x;
}

// What row r of a call wants: `n` pages at the entries from `at` on of row `row` of the table.
struct Want { int row, at, n; };

__device__ __forceinline__ Want want_of(const PagesParams& p, int r) {
  Want w{0, 0, 0};
  if (!p.source) {   // alloc
    w.row = r;
    w.at = max(0, min(p.first[r], p.max_pages));
    w.n = max(0, max(0, min(p.last[r], p.max_pages)) - w.at);
    return w;
  }
  const int s = p.source[r], t = p.target[r];   // fork: the started page of the source
  if (s < 0 || s >= p.rows || t < 0 || t >= p.rows || s == t) return w;
  const int len = max(0, p.lengths[s]);
  w.row = t;
  w.at = len >> p.shift;
  if (w.at >= p.max_pages || (len & ((1 << p.shift) - 1)) == 0) return w;
  const int page = p.table[s * p.table_stride + w.at];
  w.n = page >= 0 && page < p.num_pages ? 1 : 0;
  return w;
}

__global__ __launch_bounds__(PG_T) void pages_find_kernel(const PagesParams p) {
  __shared__ int64_t part64[PG_T / 64];
  __shared__ int part[PG_T / 64], lds_list[PG_LIST], lds_rows[PG_ROWS];
  const int tid = threadIdx.x;
  // pages wanted ahead of each row
  int* rows = p.n <= PG_ROWS ? lds_rows : p.scratch;
  int N = 0;
  for (int r0 = 0; r0 < p.n; r0 += PG_T) {
    const int r = r0 + tid;
    int64_t all;
    const int64_t before = prefix<int64_t>(r < p.n ? want_of(p, r).n : 0, part64, all);
    // (no more than there are pages)
    if (r < p.n) rows[r] = (int)min(N + before, (int64_t)p.num_pages);
    N = (int)min(N + all, (int64_t)p.num_pages);
  }
  if (N == 0 && p.source) return;
  // the first N free pages
  int* list = N <= PG_LIST ? lds_list : p.scratch + (p.n <= PG_ROWS ? 0 : p.n);
  int found = 0;
  for (int g0 = 0; g0 < p.num_pages && found < N; g0 += 4 * PG_T) {
    const int g = g0 + 4 * tid;
    int free[4], mine = 0, all;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      free[e] = g + e < p.num_pages && p.refs[min(g + e, p.num_pages - 1)] <= 0 ? 1 : 0;
      mine += free[e];
    }
    int at = found + prefix(mine, part, all);
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (free[e]) {
        if (at < N) list[at] = g + e;
        at++;
      }
    found = min(found + all, N);
  }
  __syncthreads();
  // a wave per row
  const int lane = tid & 63;
  for (int r = tid >> 6; r < p.n; r += PG_T / 64) {
    const Want w = want_of(p, r);
    const int base = rows[r];
    for (int e = lane; e < w.n; e += 64) {
      const int64_t k = (int64_t)base + e;
      const int page = k < found ? list[k] : -1;
      p.table[w.row * p.table_stride + w.at + e] = page;
      if (page >= 0) p.refs[page] = 1;
    }
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

// Fork r: the first workgroup of the row shares the whole pages (the started one is in the target's row already), all of them copy the rows of
// the started page, a head each.
__global__ __launch_bounds__(256) void pages_fork_kernel(const PagesParams p, const PagedView c, const int chunks) {
  const int r = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
  const int s = p.source[r], t = p.target[r];
  if (s < 0 || s >= p.rows || t < 0 || t >= p.rows || s == t) return;
  const int len = max(0, p.lengths[s]), whole = min(len >> p.shift, p.max_pages), rest = whole < p.max_pages ? len & ((1 << p.shift) - 1) : 0;
  const int *from = p.table + s * p.table_stride;
  int* to = p.table + t * p.table_stride;
  const int old = rest ? from[whole] : -1;
  const bool started = rest && old >= 0 && old < p.num_pages;
  if (head == 0) {
    for (int e = tid; e < p.max_pages; e += 256) {
      if (e == whole && started) continue;
      const int page = e < whole ? from[e] : -1;
      to[e] = page;
      if (page >= 0 && page < p.num_pages) atomicAdd(p.refs + page, 1);
    }
  }
  if (!started) return;
  const int fresh = to[whole];
  if (fresh < 0 || fresh >= p.num_pages || fresh == old) return;
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
// key and value.
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

// ints of scratch: rows and pages that do not fit the LDS of the search
int64_t pages_scratch_ints(int rows, int num_pages) {
  return (rows > PG_ROWS ? rows : 0) + (num_pages > PG_LIST ? num_pages : 0);
}

int launch_pages_alloc(const PagesParams& p, hipStream_t s) {
  hipLaunchKernelGGL(pages_find_kernel, dim3(1), dim3(PG_T), 0, s, p);
  return status();
}

int launch_pages_free(const PagesParams& p, hipStream_t s) {
  hipLaunchKernelGGL(pages_free_kernel, dim3((p.max_pages + 255) / 256, p.rows), dim3(256), 0, s, p);
  return status();
}

int launch_pages_fork(const PagesParams& p, const PagedView& c, int row_bytes, hipStream_t s) {
  hipLaunchKernelGGL(pages_find_kernel, dim3(1), dim3(PG_T), 0, s, p);
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
