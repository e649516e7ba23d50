// The page pool of a key-value cache (gfx950): rows take pages, are written,
// forked, trimmed and freed, and the pool is compacted, with the bookkeeping
// (page table, row lengths, a reference count per page) on the device, so
// that none of it waits for the host and all of it can be captured.
//
//   reserve  a row of length n gets the pages of tokens n .. n + n_new - 1
//   fork     a child row shares its parent's full pages (a reference more)
//            and gets a copy of the started one
//   free     a row's references are given back (trim: those of the pages that
//            neither the window nor the sinks reach any more)
//   compact  the used pages at or beyond the number of used pages move, in
//            order, into the free pages below it; tables follow
//
// Pages are taken lowest index first, rows in the order of the call, so the
// result does not depend on timing.  The bookkeeping is one workgroup's
// prefix sums over the rows and the reference counts: 4096 counts a step, and
// reserve and fork stop at the last page they need.  What takes time is the
// pages' bytes, read once and written once by workgroups that copy 16 KB runs.
// reserve and fork change nothing unless every row can be served: status[0]
// then holds the pages that were missing, status[1] the rows whose table row
// is too short.
//
// Measured: bookkeeping 5 us; compacting 453 MB (half of it read, half written)
// 86 us, 5.3 TB/s, a large copy's rate; sharing and copying 16 prompts' pages
// into 64 rows of 8 layers 17 us for 134 MB; writing 8 prompts of up to 1001
// tokens into 4 layers 15 us for 66 MB; freeing 3 us.
#include "attn_common.hpp"

namespace gdnx {

namespace {

constexpr int PT = 1024;             // threads of the bookkeeping workgroup
constexpr int PW = PT / 64;

// Exclusive prefix sum over the workgroup; *total gets the sum.  sh: PW ints.
__device__ __forceinline__ int wg_scan(int x, int* sh, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(s, off, 64);
    if (lane >= off) s += y;
  }
  __syncthreads();                   // (sh may still be read from the call before)
  if (lane == 63) sh[wave] = s;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < PW; ++w) {
    if (w < wave) base += sh[w];
    all += sh[w];
  }
  *total = all;
  return base + s - x;
}

// The first `need` free pages, in order, into list; returns how many there
// are (need, or all of the pool's).
__device__ int find_free(const int* refs, int n_pages, int need, int* list, int* sh) {
  int found = 0;
  for (int p0 = 0; p0 < n_pages && found < need; p0 += 4 * PT) {
    const int p = p0 + 4 * threadIdx.x;
    bool fr[4];
    int c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      fr[e] = p + e < n_pages && refs[p + e] == 0;
      c += fr[e];
    }
    int total;
    int at = found + wg_scan(c, sh, &total);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (fr[e]) {
        if (at < need) list[at] = p + e;
        ++at;
      }
    found += total;
  }
  return found < need ? found : need;
}

// Length of table row r, or -1 where the row does not exist or its length does not fit it.
__device__ __forceinline__ int row_length(const PagesArgs& a, int r) {
  if (r < 0 || r >= a.rows) return -1;
  const int len = a.lengths[r];
  return len >= 0 && len <= (long long)a.width * a.page ? len : -1;
}

}  // namespace

// ws: [n] first page of each row in the list, then [n_pages] free pages
__global__ void __launch_bounds__(PT) pages_reserve_kernel(PagesArgs a, int* ws) {
  __shared__ int sh[PW], s_short;
  int* offs = ws;
  int* list = ws + a.n;
  if (threadIdx.x == 0) s_short = 0;
  int need = 0;
  for (int s0 = 0; s0 < a.n; s0 += PT) {
    const int s = s0 + threadIdx.x;
    int c = 0;
    bool too_long = false;
    const int len = s < a.n ? row_length(a, a.slots[s]) : -1;
    if (len >= 0) {
      const long long want = ((long long)len + a.n_new + a.page - 1) / a.page;
      too_long = want > a.width;
      if (!too_long) c = (int)want - (len + a.page - 1) / a.page;
    }
    int total;
    const int at = wg_scan(c, sh, &total);
    if (s < a.n) offs[s] = need + at;
    if (too_long) atomicAdd(&s_short, 1);
    // (the sum is bounded by width times rows of the call, which the host keeps under 2^31)
    need += total;
  }
  const int got = find_free(a.refs, a.n_pages, need, list, sh);
  __syncthreads();
  const bool fail = got < need || s_short > 0;
  if (fail) {
    if (threadIdx.x == 0) {
      a.status[0] = need - got;
      a.status[1] = s_short;
    }
    for (int s = threadIdx.x; s < a.n; s += PT) a.start[s] = -1;
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int s = wave; s < a.n; s += PW) {
    const int r = a.slots[s], len = row_length(a, r);
    if (len < 0) {
      if (lane == 0) a.start[s] = -1;
      continue;
    }
    const int have = (len + a.page - 1) / a.page;
    const int cnt = (int)(((long long)len + a.n_new + a.page - 1) / a.page) - have, at = offs[s];
    for (int c = lane; c < cnt; c += 64) {
      const int pg = list[at + c];
      a.table[(size_t)r * a.width + have + c] = pg;
      a.refs[pg] = 1;
    }
    if (lane == 0) {
      a.start[s] = len;
      a.lengths[r] = len + a.n_new;
    }
  }
}

// slots: parents, start: children.  ws: src[n], dst[n] (-1: nothing to copy),
// offs[n], lens[n] (the parent's length; -1: no such pair), then [n] free pages
__global__ void __launch_bounds__(PT) pages_fork_kernel(PagesArgs a, int* ws) {
  __shared__ int sh[PW];
  int *src = ws, *dst = ws + a.n, *offs = ws + 2 * a.n, *lens = ws + 3 * a.n, *list = ws + 4 * a.n;
  int need = 0;
  for (int s0 = 0; s0 < a.n; s0 += PT) {
    const int s = s0 + threadIdx.x;
    int len = -1;
    if (s < a.n && a.slots[s] != a.start[s] && row_length(a, a.start[s]) == 0) len = row_length(a, a.slots[s]);
    const bool started = len > 0 && len % a.page != 0;
    int total;
    const int at = wg_scan(started, sh, &total);
    if (s < a.n) {
      lens[s] = len;
      dst[s] = -1;
      offs[s] = need + at;
    }
    need += total;
  }
  const int got = find_free(a.refs, a.n_pages, need, list, sh);
  __syncthreads();
  if (got < need) {
    if (threadIdx.x == 0) {
      a.status[0] = need - got;
      a.status[1] = 0;
    }
    for (int s = threadIdx.x; s < a.n; s += PT) lens[s] = -1;
    return;
  }
  for (int s = threadIdx.x; s < a.n; s += PT) {
    const int len = lens[s];
    if (len <= 0 || len % a.page == 0) continue;
    const int pg = list[offs[s]], full = len / a.page, from = a.table[(size_t)a.slots[s] * a.width + full];
    a.table[(size_t)a.start[s] * a.width + full] = pg;
    a.refs[pg] = 1;
    src[s] = from;
    if (from >= 0 && from < a.n_pages) dst[s] = pg;
  }
}

// A workgroup's 16 KB run of a page: 4 x 16 bytes a thread.
constexpr int kRun = 16384;
__device__ __forceinline__ void copy_run(char* dst, const char* src, long long bytes) {
  u32x4 x[4];
  const long long at = 16LL * threadIdx.x;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at + e * 4096 < bytes) x[e] = *(const u32x4*)(src + at + e * 4096);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at + e * 4096 < bytes) *(u32x4*)(dst + at + e * 4096) = x[e];
}

// Copies page src[i] onto page dst[i] in every layer of both pools; count
// from the device, or n.  The runs of the pages go round the workgroups.
__device__ __forceinline__ void copy_pages(const PagesArgs& a, const int* src, const int* dst, long long count, int wg,
                                           int n_wg) {
  const long long runs = (a.page_bytes + kRun - 1) / kRun, items = count * a.layers * 2 * runs;
  for (long long it = wg; it < items; it += n_wg) {
    const long long run = it % runs, rest = it / runs;
    const int layer = (int)(rest % a.layers);
    const long long pr = rest / a.layers, i = pr >> 1;
    const int d = dst[i], f = src[i];
    if (d < 0 || d >= a.n_pages || f < 0 || f >= a.n_pages) continue;
    char* pool = (char*)((pr & 1) ? a.v_pages : a.k_pages) + (long long)layer * a.n_pages * a.page_bytes;
    const long long at = run * kRun, left = a.page_bytes - at;
    copy_run(pool + d * a.page_bytes + at, pool + f * a.page_bytes + at, left < kRun ? left : kRun);
  }
}

__global__ void __launch_bounds__(256) pages_copy_kernel(PagesArgs a, const int* src, const int* dst) {
  copy_pages(a, src, dst, a.n, blockIdx.x, gridDim.x);
}

// The second half of a fork: the first n workgroups share a pair's full pages
// each (one workgroup's latencies, not one after the other as in the plan's
// workgroup), the others copy the started ones.
__global__ void __launch_bounds__(256) pages_share_kernel(PagesArgs a, const int* ws) {
  const int *src = ws, *dst = ws + a.n, *lens = ws + 3 * a.n;
  if ((int)blockIdx.x >= a.n) {
    copy_pages(a, src, dst, a.n, blockIdx.x - a.n, gridDim.x - a.n);
    return;
  }
  const int s = blockIdx.x, len = lens[s];
  if (len < 0) return;
  const int full = len / a.page, child = a.start[s];
  const int* tp = a.table + (size_t)a.slots[s] * a.width;
  int* tc = a.table + (size_t)child * a.width;
  for (int i = threadIdx.x; i < full; i += 256) {
    const int pg = tp[i];
    tc[i] = pg;
    if (pg >= 0 && pg < a.n_pages) atomicAdd(&a.refs[pg], 1);
  }
  if (threadIdx.x == 0) a.lengths[child] = len;
}

// ws: moves, then src[n_pages / 2], dst[n_pages / 2], then map[n_pages] (new
// index of a moved page)
__global__ void __launch_bounds__(PT) pages_plan_kernel(PagesArgs a, int* ws) {
  __shared__ int sh[PW];
  const int half = a.n_pages / 2 + 1;
  int *src = ws + 2, *dst = src + half, *map = dst + half;
  int mine = 0, used;
  for (int p = threadIdx.x; p < a.n_pages; p += PT) mine += a.refs[p] != 0;
  wg_scan(mine, sh, &used);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < a.n_pages; p0 += PT) {
    const int p = p0 + threadIdx.x, r = p < a.n_pages ? a.refs[p] : 0;
    const bool hole = p < used && r == 0, mover = p >= used && r != 0;
    // (a step holds both only where `used` falls into it)
    int th, tm;
    const int ah = wg_scan(hole, sh, &th), am = wg_scan(mover, sh, &tm);
    if (hole) dst[holes + ah] = p;
    if (mover) src[movers + am] = p;
    holes += th;
    movers += tm;
    if (p < a.n_pages && a.refs_out != a.refs) a.refs_out[p] = r;
    if (p < a.n_pages && p >= used && !mover) map[p] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += PT) {
    const int s = src[i], d = dst[i];
    map[s] = d;
    a.refs_out[d] = a.refs[s];
    a.refs_out[s] = 0;
  }
  if (threadIdx.x == 0) {
    ws[0] = movers;
    ws[1] = used;
  }
}

__global__ void __launch_bounds__(256) pages_move_kernel(PagesArgs a, const int* ws) {
  const int half = a.n_pages / 2 + 1, moves = ws[0], used = ws[1];
  const int *src = ws + 2, *dst = src + half, *map = dst + half;
  const long long n = (long long)a.rows * a.width;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int e = a.table[i];
    a.table_out[i] = e >= used && e < a.n_pages ? map[e] : e;
  }
  copy_pages(a, src, dst, moves, blockIdx.x, gridDim.x);
}

// One workgroup a row: its references given back (trim: those of the pages
// that hold no sink and end before the window of the row's last token).
__global__ void __launch_bounds__(256) pages_free_kernel(PagesArgs a) {
  const int r = a.slots[blockIdx.x];
  if (r < 0 || r >= a.rows) return;
  int* t = a.table + (size_t)r * a.width;
  int c0 = 0, c1 = a.width;
  if (a.trim) {
    const int len = a.lengths[r];
    c0 = (a.sinks + a.page - 1) / a.page;
    c1 = len > a.window ? min((len - a.window) / a.page, a.width) : 0;
  }
  for (int c = c0 + threadIdx.x; c < c1; c += 256) {
    const int pg = atomicExch(&t[c], -1);      // (a row named twice is given back once)
    if (pg >= 0 && pg < a.n_pages) atomicSub(&a.refs[pg], 1);
  }
  if (!a.trim && threadIdx.x == 0) a.lengths[r] = 0;
}

// New tokens [layers][n][n_new][Hkv][D] to their pages.  A workgroup takes
// 1024 of a layer's 16-byte units, four a thread, all loaded before the first
// is stored; units of a token follow each other, so its place is looked up
// from small numbers (one wide division a workgroup).
__global__ void __launch_bounds__(256) pages_write_kernel(PagesArgs a, unsigned per_layer) {
  const unsigned upr = a.row_bytes / 16, upt = a.Hkv * upr;    // units of a head's row, of a token
  const unsigned lk = blockIdx.x / per_layer, blk = blockIdx.x % per_layer;
  const int layer = lk >> 1;
  const long long tokens = (long long)a.n * a.n_new, first = (long long)blk * 1024;
  const long long tok0 = first / upt;
  const unsigned rem = (unsigned)(first - tok0 * upt);
  const char* from = (const char*)((lk & 1) ? a.v_new : a.k_new) + ((long long)layer * tokens * upt + first) * 16;
  char* pool = (char*)((lk & 1) ? a.v_pages : a.k_pages) + (long long)layer * a.n_pages * a.page_bytes;
  const int s0 = (int)(tok0 / a.n_new), tr0 = (int)(tok0 - (long long)s0 * a.n_new);
  u32x4 x[4];
  long long to[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned v = e * 256 + threadIdx.x, r = rem + v, dt = r / upt, u = r - dt * upt;
    to[e] = -1;
    if (tok0 + dt >= tokens) continue;
    x[e] = *(const u32x4*)(from + v * 16);
    const unsigned tt = tr0 + dt, ds = tt / (unsigned)a.n_new;
    const int s = s0 + ds, t = tt - ds * a.n_new, row = a.slots[s], st = a.start[s];
    if (row < 0 || row >= a.rows || st < 0) continue;
    const long long pos = (long long)st + t;
    if (pos >= (long long)a.width * a.page) continue;
    const int col = (int)pos / a.page, in = (int)pos - col * a.page, pg = a.table[(size_t)row * a.width + col];
    if (pg < 0 || pg >= a.n_pages) continue;
    const unsigned h = u / upr;
    to[e] = pg * a.page_bytes + ((long long)h * a.page + in) * a.row_bytes + (u - h * upr) * 16;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (to[e] >= 0) *(u32x4*)(pool + to[e]) = x[e];
}

int pages_reserve_dispatch(const PagesArgs& a, int* ws, hipStream_t stream) {
  hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(PT), 0, stream, a, ws);
  return check_launch("pages_reserve_kernel");
}

int pages_fork_dispatch(const PagesArgs& a, int* ws, hipStream_t stream) {
  hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(PT), 0, stream, a, ws);
  const int rc = check_launch("pages_fork_kernel");
  if (rc) return rc;
  const long long items = (long long)a.n * a.layers * 2 * ((a.page_bytes + kRun - 1) / kRun);
  const unsigned grid = (unsigned)(a.n + (items < 8192 ? items : 8192));
  hipLaunchKernelGGL(pages_share_kernel, dim3(grid), dim3(256), 0, stream, a, (const int*)ws);
  return check_launch("pages_share_kernel");
}

int pages_copy_dispatch(const PagesArgs& a, const int* src, const int* dst, hipStream_t stream) {
  const long long items = (long long)a.n * a.layers * 2 * ((a.page_bytes + kRun - 1) / kRun);
  const unsigned grid = (unsigned)(items < 8192 ? items : 8192);
  hipLaunchKernelGGL(pages_copy_kernel, dim3(grid), dim3(256), 0, stream, a, src, dst);
  return check_launch("pages_copy_kernel");
}

int pages_compact_dispatch(const PagesArgs& a, int* ws, hipStream_t stream) {
  hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(PT), 0, stream, a, ws);
  const int rc = check_launch("pages_plan_kernel");
  if (rc) return rc;
  hipLaunchKernelGGL(pages_move_kernel, dim3(4096), dim3(256), 0, stream, a, (const int*)ws);
  return check_launch("pages_move_kernel");
}

int pages_free_dispatch(const PagesArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(pages_free_kernel, dim3(a.n), dim3(256), 0, stream, a);
  return check_launch("pages_free_kernel");
}

int pages_write_dispatch(const PagesArgs& a, hipStream_t stream) {
  const unsigned per_layer = pages_write_groups(a);
  hipLaunchKernelGGL(pages_write_kernel, dim3(per_layer * 2 * a.layers), dim3(256), 0, stream, a, per_layer);
  return check_launch("pages_write_kernel");
}

// workgroups of one layer's keys (or values)
long long pages_write_groups(const PagesArgs& a) {
  return ((long long)a.n * a.n_new * a.Hkv * (a.row_bytes / 16) + 1023) / 1024;
}

}  // namespace gdnx
