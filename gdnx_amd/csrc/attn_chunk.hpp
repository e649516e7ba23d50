// Attention of packed new tokens over a paged cache: what its kernels share.
#pragma once
#include "attn_common.hpp"
#include "packed_rows.hpp"

namespace gdnx {

// Packed row i: its table row, tokens and positions.
struct ChunkSeq {
  int i, r, first, count, len, off;      // off: the position of its first token
  __device__ __forceinline__ void find(const ChunkAttnArgs& a, int i_, int first_, int count_) {
    i = i_;
    first = first_;
    count = count_;
    r = a.slots ? a.slots[i] : i;
    const bool there = r >= 0 && r < a.rows;
    const long long cap = (long long)a.width << a.page_log;
    len = there ? a.lengths[r] : 0;
    if (len < 0 || len > cap) len = 0;
    off = len - count;
    r = there ? r : 0;
  }
};

// Where a workgroup stands among the long rows' work: key heads fastest (a
// head's tiles share an XCD's L2 where 8 divides the heads), then the parts; a
// row's last tiles, which see most keys, first.
struct ChunkItem {
  int hk, part, item;
  __device__ __forceinline__ ChunkItem(const ChunkAttnArgs& a, int w) {
    hk = w % a.Hkv; w /= a.Hkv;
    part = w % a.parts;
    item = a.items - 1 - w / a.parts;
  }
};

// The long row and its tile of T pairs that an item is; false: none.  Up to
// kChunkListed rows, items are the long rows' tiles one after the other: the
// wave counts them through, a lane four rows, all asked for at once.  Beyond, row_item's
// places, most of which are empty where rows are short (61 single tokens on up to 8192:
// 118 us with the join by places, 111 by the list; 1000 rows on up to 1000, counted in
// steps of 64, 221, by places 198).
__device__ __forceinline__ bool chunk_item(const ChunkAttnArgs& a, int G, int T, int item, int lane, int* row, int* first,
                                           int* count, int* tile) {
  if (a.n > kChunkListed) {
    if (!row_item(a.offsets, a.n, a.N, G, T, item, lane, row, first, count, tile)) return false;
    const long long pairs = (long long)*count * G;
    return pairs > a.short_rows && (long long)*tile * T < pairs;
  }
  int o[5], c[4], t[4], sum = 0;
#pragma unroll
  for (int e = 0; e < 5; ++e) o[e] = packed_offset(a.offsets, min(4 * lane + e, a.n), a.N);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    c[e] = max(o[e + 1] - o[e], 0);                  // (none behind the last row)
    const int pairs = c[e] * G;
    t[e] = pairs > a.short_rows ? (pairs + T - 1) / T : 0;
    sum += t[e];
  }
  const int end = wave_scan(sum);
  const unsigned long long behind = __ballot(end > item);
  if (!behind) return false;
  const int l = __ffsll(behind) - 1;
  item -= __builtin_amdgcn_readlane(end - sum, l);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int tiles = __builtin_amdgcn_readlane(t[e], l);
    if (item < tiles) {
      *row = 4 * l + e;
      *first = __builtin_amdgcn_readlane(o[e], l);
      *count = __builtin_amdgcn_readlane(c[e], l);
      *tile = item;
      return true;
    }
    item -= tiles;
  }
  return false;
}

// Parts that an item of `tiles` key tiles is cut into.
__device__ __forceinline__ int chunk_parts(const ChunkAttnArgs& a, int tiles) { return max(1, min(a.parts, tiles / a.least)); }

// A short row's visible keys, counted through without a gap: the sinks, then
// from the first key that its first token's window holds on.
struct ChunkSeen {
  int lo, ns, nvis;
  __device__ __forceinline__ ChunkSeen(const ChunkAttnArgs& a, const ChunkSeq& s) {
    const int p0 = max(s.off, 0);
    lo = min(s.len, max(p0 - a.window + 1, 0));
    ns = min(a.sinks, lo);
    nvis = ns + s.len - lo;
  }
  __device__ __forceinline__ int key(int x) const { return x < ns ? x : x - ns + lo; }
};
__device__ __forceinline__ int chunk_spans(int tiles, int most) { return min(most, (tiles + 3) / 4); }

__device__ __forceinline__ float* long_out(const ChunkAttnArgs& a, int part, long long row) {
  return a.part + ((long long)part * a.N * a.Hq + row) * a.D;
}
__device__ __forceinline__ float* long_stats(const ChunkAttnArgs& a, int part, long long row) {
  const long long rows = (long long)a.N * a.Hq;
  return a.part + (long long)a.parts * rows * a.D + 2 * (part * rows + row);
}
__device__ __forceinline__ float* short_out(const ChunkAttnArgs& a, long long row, int span) {
  return a.span_part + (row * a.spans + span) * a.D;
}
__device__ __forceinline__ float* short_stats(const ChunkAttnArgs& a, long long row, int span) {
  return a.span_part + (long long)a.n * a.Hkv * kChunkShort * a.spans * a.D + 2 * (row * a.spans + span);
}

// A query from what it sees alone, by its whole wave: a lane a key for the
// scores, D / 64 columns for the sum.  In a tile that a query sees in part a
// hidden value enters its product times zero, which is NaN where the value is
// not finite, so queries whose output is not finite are formed again by this.
// Nothing of it runs while all outputs are finite.
template <typename CT, int D> struct ChunkRow {
  static constexpr int E = D / 64;
  float m, l, acc[E];
  __device__ __forceinline__ ChunkRow() : m(-INFINITY), l(0.f) {
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
  }
  // 64 more keys, the lane's being j (hidden ones among them)
  __device__ __forceinline__ void add(const ChunkAttnArgs& a, const CT* q, int r, int hk, int p, int j, int lane) {
    const int pg = j >= 0 && attn_visible(p, j, a.window, a.sinks)
                       ? a.table[(long long)r * a.width + (j >> a.page_log)] : -1;
    const bool vis = pg >= 0 && pg < a.n_pages;
    const long long at = vis ? (((long long)pg * a.Hkv + hk) << a.page_log) + (j & ((1 << a.page_log) - 1)) : 0;
    float s = 0.f;
    if (vis) {
      const CT* k = (const CT*)a.k_pages + at * D;
      for (int d = 0; d < D; ++d) s = fmaf(to_f(q[d]), to_f(k[d]), s);
    }
    s = vis ? s * (a.scale * kLog2e) : -INFINITY;
    float mx = s;
    for (int x = 32; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m - ms);
    const float pr = vis ? __builtin_amdgcn_exp2f(s - ms) : 0.f;
    float sum = pr;
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    m = mn;
    l = l * f + sum;
    for (int e = 0; e < E; ++e) acc[e] *= f;
    for (unsigned long long seen = __ballot(vis); seen; seen &= seen - 1) {
      const int key = __ffsll(seen) - 1;
      const float pk = __shfl(pr, key, 64);
      const CT* v = (const CT*)a.v_pages + __shfl(at, key, 64) * D;
      for (int e = 0; e < E; ++e) acc[e] = fmaf(pk, to_f(v[lane * E + e]), acc[e]);
    }
  }
  __device__ __forceinline__ void store(CT* y, int lane) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int e = 0; e < E; ++e) y[lane * E + e] = from_f<CT>(acc[e] * inv);
  }
  __device__ __forceinline__ void store_part(float* o, float* ml, int lane) const {
    for (int e = 0; e < E; ++e) o[lane * E + e] = acc[e];
    if (lane == 0) {
      ml[0] = m;
      ml[1] = l;
    }
  }
};

// The rows of a long item's wave in `redo` (a bit for each of its WR rows)
// formed again over what has been stored.  All of it is read and worked out
// anew from the kernel's arguments, its first and only ones, so that nothing
// is held for it in the main loop.
template <typename CT, int D, int BK, int WR> __device__ __forceinline__ void chunk_redo(unsigned redo) {
  const auto* args = (const __attribute__((address_space(4))) ChunkAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  int w = blockIdx.x, tid = opaque(threadIdx.x);
  asm volatile("" : "+s"(args), "+s"(w));
  ChunkAttnArgs a;
  __builtin_memcpy(&a, (const void*)args, sizeof(a));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.Hq / a.Hkv;
  const ChunkItem it(a, w);
  int i, first, count, tile;
  if (!chunk_item(a, G, 4 * WR, it.item, lane, &i, &first, &count, &tile)) return;
  ChunkSeq s;
  s.find(a, i, first, count);
  const RowMap rm(tile * 4 * WR, G, a.g_magic);
  const KeyTiles<BK> kt(rm.i0 + s.off, min(rm.last(4 * WR - 1), count - 1) + s.off, s.len, a.window, a.sinks);
  const int parts = chunk_parts(a, kt.count), per = (kt.count + parts - 1) / parts;
  const int t0 = it.part * per, t1 = min(kt.count, t0 + per);
  for (; redo; redo &= redo - 1) {
    int qi, h;
    rm.at(wave * WR + __ffs(redo) - 1, &qi, &h);
    if (qi >= count) continue;
    h += it.hk * G;
    const CT* q = (const CT*)a.q + (first + qi) * a.qs[0] + h * a.qs[1];
    ChunkRow<CT, D> c;
    for (int t = t0; t < t1; ++t)
      for (int jb = kt.start(t); jb < kt.start(t) + BK; jb += 64)
        c.add(a, q, s.r, it.hk, qi + s.off, lane < BK ? jb + lane : -1, lane);
    const long long row = (long long)(first + qi) * a.Hq + h;
    if (parts > 1) c.store_part(long_out(a, it.part, row), long_stats(a, it.part, row), lane);
    else c.store((CT*)a.y + row * D, lane);
  }
}

}  // namespace gdnx
