// Attention of packed new tokens over a paged key-value cache (gfx950):
// prompts' pieces, drafts and single tokens in one call.
//
//   P_j = exp(s q.k_j - lse) over the visible j,  y = sum_j P_j v_j
//
// Row i's c new tokens stand at the last c positions of its table row (its
// length counts them, and their keys and values are in their pages); the one
// at p sees key j if j <= p and p - j < window or j < sinks.  A key without a
// page is not seen.
//
// Two forms, by a row's (token, query head of the group) pairs.  Up to 32 (16 in
// float32) of them (single tokens, drafts) wait for memory: attn_chunk_short.hpp.  More
// (prompts' pieces) are tiles of 128 (64 in float32) against tiles of keys in
// LDS, as in windowed attention: attn_chunk_mfma.hip and below.  Both are in one
// launch, so that rows of both kinds share the chip; where the rows' tokens
// are is found from the offsets by the workgroups themselves, so nothing waits
// for the host.
#include "attn_chunk_short.hpp"
#include "attn_f32.hpp"

namespace gdnx {

int chunk_bf16_launch(const ChunkAttnArgs& a, unsigned groups, hipStream_t stream);

// Float32: v_mfma_f32_16x16x4_f32, a wave owns 16 rows; tiles of 32 keys by way
// of registers into LDS, double-buffered, one barrier a tile (attn_win.hip).
template <int D> __device__ __forceinline__ void chunk_long_f32(const ChunkAttnArgs& a, float* smem) {
  using T = F32Tile<D>;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.Hq / a.Hkv;
  const ChunkItem item(a, blockIdx.x);
  const int hk = item.hk;
  int si, first, count, tile;
  if (!chunk_item(a, G, 64, item.item, lane, &si, &first, &count, &tile)) return;
  ChunkSeq sq;
  sq.find(a, si, first, count);
  const int off = sq.off, len = sq.len;
  const RowMap rm(tile * 64, G, a.g_magic);
  const KeyTiles<32> kt(rm.i0 + off, min(rm.last(63), count - 1) + off, len, a.window, a.sinks);
  const int parts = chunk_parts(a, kt.count);
  if (item.part >= parts) return;
  const int per = (kt.count + parts - 1) / parts, t0 = item.part * per, t1 = min(kt.count, t0 + per);
  const int* table = a.table + (long long)sq.r * a.width;
  const int mask = (1 << a.page_log) - 1;
  const float *kb = (const float*)a.k_pages, *vb = (const float*)a.v_pages;
  int qi, qh;
  rm.at(wave * 16 + n, &qi, &qh);
  qh += hk * G;
  const int p = qi < count ? qi + off : -1;
  const int wv0 = rm.last(wave * 16) + off, last = rm.last(wave * 16 + 15);
  const int wv1 = min(last, count - 1) + off;
  const bool rows_ok = last < count && wv0 >= 0;
  f32x4 qf[T::NS];
  {
    const float* qp = (const float*)a.q + (first + (p >= 0 ? qi : 0)) * a.qs[0] + (p >= 0 ? qh : 0) * a.qs[1];
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      qf[c] = *(const f32x4*)(qp + 16 * c + 4 * g);
      if (a.scale < 0.f) qf[c] = -qf[c];
    }
  }
  const float size = fabsf(a.scale) * kLog2e, sc = size < 1e-30f ? 1e-30f : size;      // (no number stays none)
  F32Stage<D> st(tid);
  // the page of key j0 + lane of a tile, and (there) which of its 32 keys have one
  const auto page_at = [&](int it) { return table[min(kt.start(min(it, t1 - 1)) + (lane & 31), len - 1) >> a.page_log]; };
  const auto load = [&](int it, int pg) {
    const int j0 = kt.start(min(it, t1 - 1));
    const bool there = pg >= 0 && pg < a.n_pages;
    const int page = there ? pg : 0;
    st.load([&](int r, const float** x, const float** y) {
      const int c = min(r, len - 1 - j0);
      const long long at = ((((long long)__shfl(page, c) * a.Hkv + hk) << a.page_log) + ((j0 + c) & mask)) * D;
      *x = kb + at;
      *y = vb + at;
    });
    return (unsigned)__ballot(there);
  };
  f32x4 o[T::NS];
#pragma unroll
  for (int t = 0; t < T::NS; ++t) o[t] = zero4();
  float m = -INFINITY, l = 0.f;
  unsigned there = 0;
  int pg = -1;
  if (t0 < t1) {
    there = load(t0, page_at(t0));
    pg = page_at(t0 + 1);
    st.store(smem, smem + T::WORDS);
  }
  lds_barrier();
  for (int it = t0; it < t1; ++it) {
    const int j0 = kt.start(it);
    const float *sk = smem + ((it - t0) & 1) * 2 * T::WORDS, *sv = sk + T::WORDS;
    const unsigned there_next = load(it + 1, pg);
    pg = page_at(it + 2);
    if (wv0 <= wv1 && j0 <= wv1 && (j0 + 31 > wv0 - a.window || j0 < a.sinks)) {
      const bool all = rows_ok && j0 + 31 <= wv0 && (wv1 - j0 < a.window || j0 + 32 <= a.sinks) && there == ~0u;
      f32x4 s[2];
      s[0] = s[1] = zero4();
#pragma unroll
      for (int c = 0; c < T::NS; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) mma(s[u], ld_frag(sk + (16 * u + n) * T::LD + 16 * c, g), qf[c]);
      if (!all) {
        const int d = p - j0 - 4 * g, ds = a.sinks - j0 - 4 * g;
        const unsigned lv = there >> (4 * g);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = 16 * u + e;
            s[u][e] = (c <= d) & ((d - c < a.window) | (c < ds)) & (lv >> c & 1) ? s[u][e] : -INFINITY;
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * sc;
      if (__any(mx > m + 8.f)) {             // (raised by steps of 2^8)
        const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int t = 0; t < T::NS; ++t) o[t] *= f;
      }
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], sc, -ms));
          l += s[u][e];
        }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t = 0; t < T::NS; ++t) mma(o[t], ld_cols<T::LD>(sv, 16 * u, 16 * t + n, g), s[u]);
    }
    float* next = smem + ((it - t0 + 1) & 1) * 2 * T::WORDS;
    st.store(next, next + T::WORDS);
    lds_barrier();
    there = there_next;
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (p < 0) {                              // a row that sees nothing: 0 times a value that is not finite is NaN
#pragma unroll
    for (int t = 0; t < T::NS; ++t) o[t] = zero4();
  }
  // rows of the wave whose output is not finite (0 times it is NaN)
  float rest = 0.f;
#pragma unroll
  for (int t = 0; t < T::NS; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) rest = fmaf(o[t][e], 0.f, rest);
  const unsigned long long bad = __ballot(rest != 0.f);
  const unsigned redo = (unsigned)(bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffffu;
  const long long r = (long long)(first + qi) * a.Hq + qh;
  if (qi < count && parts > 1) {
    float* po = long_out(a, item.part, r) + 4 * g;
#pragma unroll
    for (int t = 0; t < T::NS; ++t) *(f32x4*)(po + 16 * t) = o[t];
    if (g == 0) {
      float* ml = long_stats(a, item.part, r);
      ml[0] = m;
      ml[1] = l;
    }
  } else if (qi < count) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < T::NS; ++t) *(f32x4*)((float*)a.y + r * D + 16 * t + 4 * g) = o[t] * inv;
  }
  if (redo) {
    __builtin_amdgcn_s_waitcnt(0x0070);             // (the wave's own stores come first)
    chunk_redo<float, D, 32, 16>(redo);
  }
}

template <int D> __global__ void __launch_bounds__(256, 2) chunk_f32_kernel(ChunkAttnArgs a) {
  constexpr int WORDS = F32Tile<D>::WORDS;
  __shared__ __attribute__((aligned(16))) float smem[4 * WORDS];       // two buffers of K, V
  __shared__ ChunkShortShared<float> sh;
  const int n_long = a.items * a.parts * a.Hkv;
  if ((int)blockIdx.x < n_long) chunk_long_f32<D>(a, smem);
  else chunk_short<float, D>(a, blockIdx.x - n_long, [&](int v) { return (char*)(smem + v * WORDS); }, sh);
}

// Running joins of (maximum, sum, output) triples.
struct ChunkJoin {
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float m2, float l2, const f32x4& x) {
    const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ms), g = __builtin_amdgcn_exp2f(m2 - ms);
    l = l * f + l2 * g;
    acc = acc * f + x * g;
    m = mn;
  }
  // every `step`-th of n, four asked for at a time (the last again where there are no four)
  template <typename S, typename O>
  __device__ __forceinline__ void take(int n, int from, int step, const S& stats, const O& out) {
    for (int x0 = from; x0 < n; x0 += 4 * step) {
      float ml[4][2];
      f32x4 o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int x = min(x0 + e * step, n - 1);
        ml[e][0] = stats(x)[0];
        ml[e][1] = stats(x)[1];
        o[e] = *(const f32x4*)out(x);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x0 + e * step < n) add(ml[e][0], ml[e][1], o[e]);
    }
  }
  template <typename CT> __device__ __forceinline__ void store(CT* y) const {
    const f32x4 o = acc * (l == 0.f ? 0.f : 1.f / l);
    st4(y, o[0], o[1], o[2], o[3]);
  }
};

// Parts and spans joined in order.  Long rows: D / 4 threads a pair, one pair
// after the other only where the items are many (200 tokens on 16384 in 16 parts:
// four pairs 39 us, one 7).  Short rows: so many groups of D / 4 threads a pair that each has about four
// spans; with many rows a workgroup takes all pairs of one (256 single tokens, a
// workgroup a possible pair: 54 us, most of it workgroups without work).
template <typename CT, int D> __global__ void __launch_bounds__(256) chunk_join_kernel(ChunkAttnArgs a) {
  constexpr int V = D / 4, NG = 256 / V, R = sizeof(CT) == 2 ? 128 : 64, BK = R / 2;
  __shared__ __attribute__((aligned(16))) float s_acc[NG][D];
  __shared__ float s_m[NG], s_l[NG];
  const int G = a.Hq / a.Hkv, grp = threadIdx.x / V, d = 4 * (threadIdx.x % V), lane = threadIdx.x & 63;
  int w = blockIdx.x;
  const int n_long = a.parts > 1 ? a.items * a.Hkv * a.join_split : 0;
  ChunkSeq s;
  if (w < n_long) {
    const int q0 = w % a.join_split * (R / a.join_split) + grp, q1 = q0 - grp + R / a.join_split; w /= a.join_split;
    const int hk = w % a.Hkv;
    int i, first, count, tile;
    if (!chunk_item(a, G, R, w / a.Hkv, lane, &i, &first, &count, &tile)) return;
    s.find(a, i, first, count);
    const RowMap rm(tile * R, G, a.g_magic);
    const KeyTiles<BK> kt(rm.i0 + s.off, min(rm.last(R - 1), count - 1) + s.off, s.len, a.window, a.sinks);
    const int parts = chunk_parts(a, kt.count);
    if (parts == 1) return;                        // written by its workgroup
    for (int q = q0; q < q1; q += NG) {
      int qi, h;
      rm.at(q, &qi, &h);
      if (qi >= count) return;
      const long long row = (long long)(first + qi) * a.Hq + hk * G + h;
      ChunkJoin j;
      j.take(parts, 0, 1, [&](int x) { return long_stats(a, x, row); }, [&](int x) { return long_out(a, x, row) + d; });
      j.store((CT*)a.y + row * D + d);
    }
    return;
  }
  w -= n_long;
  // `share` groups of threads take a pair's spans, 256 / V / share pairs a workgroup at a time
  const int share = min(a.join_share, NG), step = NG / share, blocks = a.join_blocks;
  const int block = w % blocks; w /= blocks;
  const int hk = w % a.Hkv, i = w / a.Hkv;
  const int first = packed_offset(a.offsets, i, a.N), count = packed_offset(a.offsets, i + 1, a.N) - first;
  if (count <= 0 || (long long)count * G > a.short_rows || block * step >= count * G) return;
  s.find(a, i, first, count);
  const ChunkSeen see(a, s);
  constexpr int BT = FragT<CT>::KSTEP;
  const int spans = chunk_spans((see.nvis + BT - 1) / BT, a.spans);
  if (spans <= 1) return;                          // written by its workgroup
  for (int q0 = block * step; q0 < count * G; q0 += blocks * step) {
    const int q = q0 + grp / share, part = grp % share;
    const long long row = ((long long)i * a.Hkv + hk) * kChunkShort + q;
    ChunkJoin j;
    if (q < count * G) j.take(spans, part, share, [&](int x) { return short_stats(a, row, x); },
                              [&](int x) { return short_out(a, row, x) + d; });
    if (share > 1) {
      __syncthreads();
      *(f32x4*)&s_acc[grp][d] = j.acc;
      if (d == 0) {
        s_m[grp] = j.m;
        s_l[grp] = j.l;
      }
      __syncthreads();
      if (part == 0)
        for (int x = 1; x < share; ++x) j.add(s_m[grp + x], s_l[grp + x], *(const f32x4*)&s_acc[grp + x][d]);
    }
    if (part == 0 && q < count * G) j.store((CT*)a.y + ((long long)(first + q / G) * a.Hq + hk * G + q % G) * D + d);
  }
}

// How the rows share the work.  Their lengths are on the device, so the
// numbers of workgroups come from the batch's size and from the longest row that the
// table can hold (or the window); what a row does not need ends at once.
//
// Long rows' keys are cut into parts where the tiles do not give every CU its
// two workgroups (one row), or twice that (several, whose lengths differ, so that
// parts level out: three pieces up to 1024 on up to 8192 tokens 265 us with the join uncut,
// 220 in two, 200 in three, 204 in four), but into no more than 4096 workgroups, many of which have
// no work where rows are short (256 single tokens, rows by places: 402 us, 418 with 11600 of them).
// A part has four tiles at least, eight where the tiles are many already; in us with the
// join, eight / four: 8 x 9 tokens on 2000, 16/4 heads, 37 / 25; 12 float32 rows with a
// window of 512 29 / 21; 4 x 512 on 500 46 / 50.
void chunk_attn_plan(ChunkAttnArgs& a) {
  const long long G = a.Hq / a.Hkv, R = a.dtype == GDNX_DTYPE_BF16 ? 128 : 64, pairs = a.N * G;
  long long keys = (long long)a.width << a.page_log;
  // A single row too may hold fewer tokens than the batch has places: one on 30001 cached takes 22 us alone and 23 in a batch
  // of 2048 (515 where a single row went the long way whatever it held).  Rows are all short if all tokens make but one short row.
  const int short_pairs = a.short_rows = chunk_short_pairs(a.dtype == GDNX_DTYPE_BF16 ? 2 : 4);
  a.items = 0;
  a.parts = a.least = 1;
  if (pairs > a.short_rows) {
    const long long win = (long long)a.window + a.sinks + R / G + 1, span = win < keys ? win : keys;
    const long long most = pairs / (a.short_rows + 1), rows = a.n < most ? a.n : most;      // long rows there can be
    a.items = (int)(pairs / R + (a.n > kChunkListed ? a.n : rows));
    const long long tiles = ((pairs + R - 1) / R + (rows - 1) / 2) * a.Hkv;
    long long parts = (a.n == 1 ? 512 : 1024) / (tiles ? tiles : 1);
    if (parts > 4096 / ((long long)a.items * a.Hkv)) parts = 4096 / ((long long)a.items * a.Hkv);
    a.least = tiles > 192 ? 8 : 4;
    if (parts > span / (R / 2) / a.least) parts = span / (R / 2) / a.least;
    a.parts = parts < 1 ? 1 : parts > 64 ? 64 : (int)parts;
    a.join_split = (long long)a.items * a.Hkv >= 256 ? 4 : (int)(R * a.D / 1024);      // workgroups an item
  }
  const long long win = (long long)a.window + a.sinks + kChunkShort;
  a.spans = paged_attn_spans(a.n, a.Hkv, a.Hkv, win < keys ? win : keys, a.dtype);
  const int groups = 1024 / a.D;                       // of a join's workgroup
  a.join_share = 1;
  while (a.join_share < groups && 4 * a.join_share < a.spans) a.join_share *= 2;
  a.join_blocks = (long long)a.n * a.Hkv >= 512 ? 1 : (short_pairs + groups / a.join_share - 1) / (groups / a.join_share);
}

template <typename CT, int D> static int join(const ChunkAttnArgs& a, hipStream_t stream) {
  const long long groups = (a.parts > 1 ? (long long)a.items * a.Hkv * a.join_split : 0) +
                           (a.spans > 1 ? (long long)a.n * a.Hkv * a.join_blocks : 0);
  if (groups == 0) return GDNX_OK;
  hipLaunchKernelGGL((chunk_join_kernel<CT, D>), dim3((unsigned)groups), dim3(256), 0, stream, a);
  return check_launch("chunk_join_kernel");
}

int chunk_attn_dispatch(const ChunkAttnArgs& a, hipStream_t stream) {
  const unsigned groups = (unsigned)((long long)a.items * a.parts * a.Hkv + (long long)a.n * a.Hkv * a.spans);
  int rc;
  if (a.dtype == GDNX_DTYPE_BF16) {
    if ((rc = chunk_bf16_launch(a, groups, stream))) return rc;
    return a.D == 128 ? join<bf16, 128>(a, stream) : join<bf16, 64>(a, stream);
  }
  if (a.D == 128) hipLaunchKernelGGL((chunk_f32_kernel<128>), dim3(groups), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((chunk_f32_kernel<64>), dim3(groups), dim3(256), 0, stream, a);
  if ((rc = check_launch("chunk_f32_kernel"))) return rc;
  return a.D == 128 ? join<float, 128>(a, stream) : join<float, 64>(a, stream);
}

}  // namespace gdnx
