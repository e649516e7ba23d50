// The page pool of a key-value cache (gfx950): rows take pages, are written,
// forked, trimmed and freed, and the pool is compacted, with the bookkeeping
// (page table, row lengths, a reference count per page) on the device, so
// that none of it waits for the host and all of it can be captured.
//
//   reserve  a row of length n gets the pages of tokens n .. n + n_new - 1
//            (for pages that its entries still name, those are given back)
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
#include "packed_rows.hpp"

namespace gdnx {

namespace {

constexpr int PT = 1024;             // threads of the bookkeeping workgroup
constexpr int PW = PT / 64;

// Exclusive prefix sum over the workgroup; *total gets the sum.  sh: PW of them.
template <typename T> __device__ __forceinline__ T wg_scan(T x, T* sh, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T s = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(s, off, 64);
    if (lane >= off) s += y;
  }
  __syncthreads();                   // (sh may still be read from the call before)
  if (lane == 63) sh[wave] = s;
  __syncthreads();
  T base = 0, all = 0;
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

// Exclusive prefix sums over the workgroup of x and of y, and the sums.  Its
// barriers wait for LDS alone: stores to memory stay in flight.
template <typename T> __device__ __forceinline__ void wg_scan2(T* x, int* y, T* shx, int* shy, T* sumx, int* sumy) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T sx = wave_scan(*x);
  const int sy = wave_scan(*y);
  lds_barrier();                     // (what the call before left may still be read)
  if (lane == 63) {
    shx[wave] = sx;
    shy[wave] = sy;
  }
  lds_barrier();
  T bx = 0, ax = 0;
  int by = 0, ay = 0;
#pragma unroll
  for (int w = 0; w < PW; ++w) {
    const T ex = shx[w];
    const int ey = shy[w];
    if (w < wave) {
      bx += ex;
      by += ey;
    }
    ax += ex;
    ay += ey;
  }
  *x = bx + sx - *x;
  *y = by + sy - *y;
  *sumx = ax;
  *sumy = ay;
}

// find_free for many pages: four runs of 4 PT counts a step, whose prefix sums
// are the 16-bit parts of two (45 thousand of 65536 pages: the reserve takes 16.7 us;
// by single runs 33, with barriers that wait for the list's stores 20).  For
// up to 4 PT pages single runs, which look at no more of the pool than they need
// (20 rows, 30000 pages: 5.2 us, by four runs 5.8).
__device__ int find_many_free(const int* refs, int n_pages, int need, int* list, int* sh, int* sh2) {
  int found = 0;
  for (int p0 = 0; p0 < n_pages && found < need; p0 += 16 * PT) {
    unsigned fr = 0;
    int c[2] = {0, 0};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + 4 * (r * PT + (int)threadIdx.x);
      int x[4] = {1, 1, 1, 1};
      if (p + 4 <= n_pages) {
        __builtin_memcpy(x, refs + p, sizeof(x));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (p + e < n_pages) x[e] = refs[p + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        fr |= (x[e] == 0 ? 1u : 0u) << (4 * r + e);
        c[r >> 1] += (x[e] == 0) << (16 * (r & 1));
      }
    }
    int total[2];
    wg_scan2(&c[0], &c[1], sh, sh2, &total[0], &total[1]);       // (a run's sum is 4 PT at most)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      int at = found + (c[r >> 1] >> (16 * (r & 1)) & 0xffff);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (fr >> (4 * r + e) & 1) {
          if (at < need) list[at] = p0 + 4 * (r * PT + (int)threadIdx.x) + e;
          ++at;
        }
      found += total[r >> 1] >> (16 * (r & 1)) & 0xffff;
    }
  }
  return found < need ? found : need;
}

// Length of table row r, or -1 where the row does not exist or its length does not fit it.
__device__ __forceinline__ int row_length(const PagesArgs& a, int r) {
  if (r < 0 || r >= a.rows) return -1;
  const int len = a.lengths[r];
  return len >= 0 && len <= (long long)a.width * a.page ? len : -1;
}

// A taken page into a row's entry.  Where the caller has lowered the row's
// length the entry may still name the page that it had: that one is given back.
__device__ __forceinline__ void put_page(int* entry, int pg, int* refs, int n_pages) {
  const int old = *entry;
  *entry = pg;
  refs[pg] = 1;
  if (old >= 0 && old < n_pages) atomicSub(&refs[old], 1);
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
    for (int c = lane; c < cnt; c += 64) put_page(&a.table[(size_t)r * a.width + have + c], list[at + c], a.refs, a.n_pages);
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
    const int at = wg_scan((int)started, sh, &total);
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
    put_page(&a.table[(size_t)a.start[s] * a.width + full], pg, a.refs, a.n_pages);
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
    const int pg = tp[i], old = tc[i];
    tc[i] = pg;
    if (pg >= 0 && pg < a.n_pages) atomicAdd(&a.refs[pg], 1);
    if (old >= 0 && old < a.n_pages) atomicSub(&a.refs[old], 1);      // (put_page)
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
    const int ah = wg_scan((int)hole, sh, &th), am = wg_scan((int)mover, sh, &tm);
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

// ---- packed rows of unlike lengths ----
// The rows' tokens packed one after the other, and their pages: first a
// workgroup's prefix sums over the rows (as in a reserve), then a thread for
// every page that was taken and one for every packed token.
// ws: [n + 1] first page of each row in the list (its end: how many there are), then [n_pages] free pages
__global__ void __launch_bounds__(PT) pages_reserve_packed_kernel(PagesPackedArgs a, int* ws) {
  __shared__ int sh[PW], sh2[PW], s_bad;
  __shared__ long long sl[PW];
  int* offs = ws;
  int* list = ws + a.n + 1;
  if (threadIdx.x == 0) s_bad = 0;
  PagesArgs pool{};
  pool.lengths = a.lengths; pool.rows = a.rows; pool.width = a.width; pool.page = a.page;
  long long tokens = 0;
  int need = 0;
  for (int s0 = 0; s0 < a.n; s0 += PT) {
    const int s = s0 + threadIdx.x;
    const int add = s < a.n ? max(a.n_new[s], 0) : 0, len = s < a.n ? row_length(pool, a.slots[s]) : -1;
    bool bad = false;
    int at = 0, total;                       // pages
    if (len >= 0) {
      const long long want = ((long long)len + add + a.page - 1) / a.page;
      if (want > a.width) bad = true;
      else at = (int)want - (len + a.page - 1) / a.page;
    }
    long long off = add, sum;
    wg_scan2(&off, &at, sl, sh, &sum, &total);
    off += tokens;
    tokens += sum;
    bad = bad || (s < a.n && off + add > a.N);       // its last token lies behind the batch
    if (s < a.n) {
      offs[s] = need + at;
      a.offsets[s] = (int)min(off, (long long)a.N);
      a.start[s] = len;
    }
    if (bad) atomicAdd(&s_bad, 1);
    need += total;                           // (at most width times rows, which the host keeps under 2^31)
  }
  const int got = need > 4 * PT ? find_many_free(a.refs, a.n_pages, need, list, sh, sh2)
                                : find_free(a.refs, a.n_pages, need, list, sh);
  __syncthreads();
  const bool fail = got < need || s_bad > 0;
  if (threadIdx.x == 0) {
    offs[a.n] = fail ? 0 : need;
    a.offsets[a.n] = fail ? 0 : (int)tokens;
    if (fail) {
      a.status[0] = need - got;
      a.status[1] = s_bad;
    }
  }
  for (int s = threadIdx.x; s < a.n; s += PT) {
    if (fail) {
      a.offsets[s] = 0;
      a.start[s] = -1;
    } else if (a.start[s] >= 0) {
      a.lengths[a.slots[s]] = a.start[s] + max(a.n_new[s], 0);
    }
  }
}

__global__ void __launch_bounds__(256) pages_place_kernel(PagesPackedArgs a, const int* ws) {
  const int *offs = ws, *list = ws + a.n + 1;
  const int lane = threadIdx.x & 63, lg = __ffs(a.page) - 1, mask = a.page - 1;
  const int base = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 256 + (threadIdx.x & ~63u))), u = base + lane;
  // the last row that starts at or before u; a wave's 64 are often of one
  const auto row_of = [&](const int* starts) {
    int lo = max(wave_find(a.n, base, lane, [&](int i) { return (long long)starts[i]; }), 0), hi = a.n - 1;
    if (starts[lo + 1] > base + 63) return lo;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (starts[mid] <= u) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  const int taken = offs[a.n], tokens = a.offsets[a.n];
  if (base < taken) {
    const int s = row_of(offs);
    if (u < taken) {
      const int col = ((a.start[s] + mask) >> lg) + u - offs[s];
      put_page(&a.table[(size_t)a.slots[s] * a.width + col], list[u], a.refs, a.n_pages);
    }
  }
  if (base >= a.N) return;
  int pos = -1, place = -1;
  if (base < tokens) {
    const int s = row_of(a.offsets), st = a.start[s];
    if (u < tokens && st >= 0) {
      pos = st + u - a.offsets[s];
      const int col = pos >> lg, had = (st + mask) >> lg;
      const int pg = col < had ? a.table[(size_t)a.slots[s] * a.width + col] : list[offs[s] + col - had];
      if (pg >= 0 && pg < a.n_pages) place = (pg << lg) + (pos & mask);
    }
  }
  if (u < a.N) {
    a.positions[u] = pos;
    a.places[u] = place;
  }
}

// Packed keys and values to their places.  As pages_write_kernel: 1024 of a
// layer's 16-byte units a workgroup, four a thread, all loaded before the first
// is stored.
__global__ void __launch_bounds__(256) pages_put_kernel(PagesPutArgs a, unsigned per_layer) {
  const unsigned upr = a.row_bytes / 16, upt = a.Hkv * upr;    // units of a head's row, of a token
  const unsigned lk = blockIdx.x / per_layer, blk = blockIdx.x % per_layer;
  const int layer = lk >> 1;
  const long long first = (long long)blk * 1024;
  const int tok0 = (int)(first / upt);
  const unsigned rem = (unsigned)(first - (long long)tok0 * upt);
  const bool val = lk & 1;
  const long long st = val ? a.vs[1] : a.ks[1], sh = val ? a.vs[2] : a.ks[2];
  const char* from = (const char*)(val ? a.v_new : a.k_new) + layer * (val ? a.vs[0] : a.ks[0]);
  char* pool = (char*)(val ? a.v_pages : a.k_pages) + (long long)layer * a.n_pages * a.page_bytes;
  u32x4 x[4];
  long long to[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned r = rem + e * 256 + threadIdx.x, dt = r / upt, u = r - dt * upt, h = u / upr;
    const long long t = (long long)tok0 + dt;
    to[e] = -1;
    if (t >= a.N) continue;
    const int place = a.places[t];
    if (place < 0) continue;
    const int pg = place / a.page, in = place - pg * a.page;
    if (pg >= a.n_pages) continue;
    x[e] = *(const u32x4*)(from + t * st + h * sh + (u - h * upr) * 16);
    to[e] = pg * a.page_bytes + ((long long)h * a.page + in) * a.row_bytes + (u - h * upr) * 16;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (to[e] >= 0) *(u32x4*)(pool + to[e]) = x[e];
}

int pages_reserve_packed_dispatch(const PagesPackedArgs& a, int* ws, hipStream_t stream) {
  hipLaunchKernelGGL(pages_reserve_packed_kernel, dim3(1), dim3(PT), 0, stream, a, ws);
  const int rc = check_launch("pages_reserve_packed_kernel");
  if (rc) return rc;
  // pages that can be taken: a started page for every row besides those that the tokens fill
  const long long full = (long long)a.N / a.page + a.n, most = full < a.n_pages ? full : a.n_pages;
  const long long threads = most > a.N ? most : a.N;
  if (threads == 0) return GDNX_OK;
  hipLaunchKernelGGL(pages_place_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a,
                     (const int*)ws);
  return check_launch("pages_place_kernel");
}

long long pages_put_groups(const PagesPutArgs& a) {
  return ((long long)a.N * a.Hkv * (a.row_bytes / 16) + 1023) / 1024;
}

int pages_put_dispatch(const PagesPutArgs& a, hipStream_t stream) {
  const unsigned per_layer = (unsigned)pages_put_groups(a);
  hipLaunchKernelGGL(pages_put_kernel, dim3(per_layer * 2 * a.layers), dim3(256), 0, stream, a, per_layer);
  return check_launch("pages_put_kernel");
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
