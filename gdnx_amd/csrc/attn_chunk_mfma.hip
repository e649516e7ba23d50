// Attention of packed new tokens over a paged cache for bf16 (gfx950).  Rules
// and shares of the work in attn_chunk.hip.
#include "attn_chunk_short.hpp"
#include "attn_tiles.hpp"

namespace gdnx {

namespace {

// 64 tokens of a paged row straight into LDS (TileLoad, with the rows' places
// from the table): lane x holds the page of key j0 + x, or of the last one.  An
// instruction fills `ROWS` tokens, which lie in one page where it has so many:
// its place is then a scalar, 32-bit offsets are the lanes'.  (By lane
// exchanges throughout, as SMALL pages need it, the kernel took 673 us for 2048
// tokens on 30001 where scalar places took 580, in turn on one card.)
template <int D, bool SMALL> struct PagedTileLoad {
  using T = Tile<D>;
  static constexpr int N = 64 * T::UPR / 256, STEP = 256 / T::UPR, ROWS = 64 / T::UPR;
  unsigned row, u;
  int wave, mask;
  __device__ __forceinline__ PagedTileLoad(int tid, int wave_, int log) : row(tid / T::UPR), wave(wave_), mask((1 << log) - 1) {
    u = ((tid % T::UPR) ^ T::swz(row)) * 16;
  }
  __device__ __forceinline__ void load(char* tk, const char* k, char* tv, const char* v, long long page, int j0, int last) const {
    typedef __attribute__((address_space(1))) void* G;
    typedef __attribute__((address_space(3))) void* L;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = min((int)row + i * STEP, last), x = i * STEP + wave * ROWS;
      const unsigned in = ((j0 + r) & mask) * T::RB + u;
      long long at;
      if constexpr (SMALL) at = __shfl(page, r);
      else at = (long long)__builtin_amdgcn_readlane((int)(page >> 32), x) << 32 | (unsigned)__builtin_amdgcn_readlane((int)page, x);
      __builtin_amdgcn_global_load_lds((G)(k + at + in), (L)(tk + i * 4096 + wave * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((G)(v + at + in), (L)(tv + i * 4096 + wave * 1024), 16, 0, 0);
    }
  }
};

}  // namespace

// Long rows: a workgroup of four waves takes 128 (token, query head of the
// group) pairs of one key head, heads fastest, a wave 32 of them, over one part
// of their keys; tiles of 64 keys, double-buffered, one barrier a tile.  The
// form of win_fwd_bf16_kernel (attn_win_mfma.hip): S^T = K Q^T, a lane holding 32
// scores of one row; O^T += V^T P^T.  The page of a tile's keys is looked up
// two tiles ahead.
//
// P is rounded to bf16 for the second product, as there (its sum is of the values
// before): y is 2.0e-3 to 2.3e-3 from 64 bits, of which 1.7e-3 are its own rounding.
// A third product of what that rounding leaves over, which short rows have for
// nothing (they wait for memory), takes the whole call from 537 to 716 us for 2048
// tokens on 30001, 225 to 258 for three pieces beside 61 single tokens, and 107 to 134 for
// 4096 tokens on none.
template <int D, bool SMALL>
__device__ __forceinline__ void chunk_long(const ChunkAttnArgs& a, char (&k0)[64 * Tile<D>::RB], char (&v0)[64 * Tile<D>::RB],
                                           char (&k1)[64 * Tile<D>::RB], char (&v1)[64 * Tile<D>::RB]) {
  using T = Tile<D>;
  constexpr int BK = 64;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv;
  const ChunkItem item(a, blockIdx.x);
  const int hk = item.hk;
  int si, first, count, tile;
  if (!chunk_item(a, G, 128, item.item, lane, &si, &first, &count, &tile)) return;
  ChunkSeq sq;
  sq.find(a, si, first, count);
  const int off = sq.off, len = sq.len;
  const RowMap rm(tile * 128, G, a.g_magic);
  // positions of the workgroup's rows
  const int wg0 = rm.i0 + off, wg1 = min(rm.last(127), count - 1) + off;
  const KeyTiles<BK> kt(wg0, wg1, len, a.window, a.sinks);
  const int parts = chunk_parts(a, kt.count);
  if (item.part >= parts) return;
  const int per = (kt.count + parts - 1) / parts, t0 = item.part * per, t1 = min(kt.count, t0 + per);
  const int* table = a.table + (long long)sq.r * a.width;
  const long long page_bytes = ((long long)a.Hkv * T::RB) << a.page_log;
  const char* kb = (const char*)a.k_pages + (((long long)hk * T::RB) << a.page_log);
  const char* vb = (const char*)a.v_pages + (((long long)hk * T::RB) << a.page_log);

  // the wave's rows
  int qi, qh;
  rm.at(wave * 32 + n, &qi, &qh);
  qh += hk * G;
  const int p = qi < count ? qi + off : -1;
  bf16x8 qf[T::NS];
  {
    const bf16* qp = (const bf16*)a.q + (first + (p >= 0 ? qi : 0)) * a.qs[0] + (p >= 0 ? qh : 0) * a.qs[1];
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      qf[c] = *(const bf16x8*)(qp + 16 * c + 8 * h);
      if (a.scale < 0.f) qf[c] = -qf[c];
    }
  }
  const float size = fabsf(a.scale) * kLog2e, sc = size < 1e-30f ? 1e-30f : size;      // (no number stays none)
  const int wv0 = rm.last(wave * 32) + off, wv1 = min(rm.last(wave * 32 + 31), count - 1) + off;
  const bool rows_ok = rm.last(wave * 32 + 31) < count && wv0 >= 0;

  f32x16 o[T::ND];
#pragma unroll
  for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  float m = -INFINITY, l = 0.f;

  const LaneMap<D> lm(lane);
  const PagedTileLoad<D, SMALL> tl(tid, wave, a.page_log);
  const auto page_at = [&](int it) { return table[min(kt.start(min(it, t1 - 1)) + lane, len - 1) >> a.page_log]; };
  // asks for a tile; which of its keys are there
  const auto load = [&](char* tk, char* tv, int it, int pg) {
    const int j0 = kt.start(min(it, t1 - 1));
    const bool there = pg >= 0 && pg < a.n_pages;
    tl.load(tk, kb, tv, vb, (there ? pg : 0) * page_bytes, j0, len - 1 - j0);
    return __ballot(there);
  };
  const auto tile_step = [&](const char* tk, const char* tv, int it, unsigned long long there) {
    const int j0 = kt.start(it);
    // whether the wave sees anything of the tile, and all of it
    const bool some = it < t1 && wv0 <= wv1 && j0 <= wv1 && (j0 + BK - 1 > wv0 - a.window || j0 < a.sinks);
    if (!some) return;
    // Matrix instructions go before the other wave's vector instructions, and a tile's exponentials are through before its
    // second products, so that the two waves of a SIMD take turns.  The kernel in us, in turn on one card (others take
    // 540 to 576 for the first): 2048 tokens on 30001 582 -> 555, 1024 on 8192 92 -> 90, 8192 on 8192 777 -> 774, 4096 on
    // none 97 -> 102 (16/4 heads, d = 128).
    __builtin_amdgcn_s_setprio(1);
    const bool all = rows_ok && j0 + BK - 1 <= wv0 && (wv1 - j0 < a.window || j0 + BK <= a.sinks) && there == ~0ULL;
    f32x16 s[2];
    s[0] = s[1] = zero16();
    {                                      // (operands read two ahead: left alone, right before their use)
      bf16x8 fk[T::NS][2];
      const auto fetch = [&](int c) {
        fk[c][0] = lm.row(tk, c);
        fk[c][1] = lm.row(tk + 32 * T::RB, c);
      };
      fetch(0);
      fetch(1);
#pragma unroll
      for (int c = 0; c < T::NS; ++c) {
        __builtin_amdgcn_sched_barrier(0);
        if (c + 2 < T::NS) fetch(c + 2);
        mma32(s[0], fk[c][0], qf[c]);
        mma32(s[1], fk[c][1], qf[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if (!all) {
      const int d = p - j0 - 4 * h, ds = a.sinks - j0 - 4 * h;
      const unsigned long long lv = there >> (4 * h);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = 32 * u + 8 * (e >> 2) + (e & 3);
          s[u][e] = (c <= d) & ((d - c < a.window) | (c < ds)) & (lv >> c & 1) ? s[u][e] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
    mx = half_max(mx) * sc;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= f;
#pragma unroll
      for (int t = 0; t < T::ND; ++t) o[t] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], sc, -ms));
        sum += s[u][e];
      }
    l += sum;
    asm volatile("" : "+v"(s[0]), "+v"(s[1]));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 pf = acc_frag32(s[u], c);
#pragma unroll
        for (int t = 0; t < T::ND; ++t) mma32(o[t], lm.cols(tv + (32 * u + 16 * c) * T::RB, t), pf);
      }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  };
  if (t0 < t1) {
    unsigned long long there0 = load(k0, v0, t0, page_at(t0)), there1;
    int pg = page_at(t0 + 1);
    loads_done_barrier();
    for (int it = t0; it < t1; it += 2) {
      there1 = load(k1, v1, it + 1, pg);
      pg = page_at(it + 2);
      tile_step(k0, v0, it, there0);
      loads_done_barrier();
      there0 = load(k0, v0, it + 2, pg);
      pg = page_at(it + 3);
      tile_step(k1, v1, it + 1, there1);
      loads_done_barrier();
    }
  }
  l = half_sum(l);
  if (p < 0) {                             // a row that sees nothing: 0 times a value that is not finite is NaN
#pragma unroll
    for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  }
  // rows of the wave whose output is not finite (0 times it is NaN)
  float rest = 0.f;
#pragma unroll
  for (int t = 0; t < T::ND; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) rest = fmaf(o[t][e], 0.f, rest);
  const unsigned long long bad = __ballot(rest != 0.f);
  const unsigned redo = (unsigned)(bad | bad >> 32);
  if (parts > 1) {                         // a part of the keys: unnormalised, joined by chunk_join_kernel
    if (qi < count) {
      const long long r = (long long)(first + qi) * a.Hq + qh;
      float* po = long_out(a, item.part, r) + 4 * h;
#pragma unroll
      for (int t = 0; t < T::ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(po + 32 * t + 8 * i) = (f32x4){o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
      if (h == 0) {
        float* ml = long_stats(a, item.part, r);
        ml[0] = m;
        ml[1] = l;
      }
    }
    if (redo) {
      __builtin_amdgcn_s_waitcnt(0x0070);           // (the wave's own stores come first)
      chunk_redo<bf16, D, BK, 32>(redo);
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  // the output by way of LDS, so that whole rows are stored
  lm.put((wave < 2 ? k0 : v0) + (wave & 1) * 32 * T::RB, o, inv);
  __syncthreads();
  bf16* yb = (bf16*)a.y + (long long)first * a.Hq * D;
#pragma unroll
  for (int u = tid; u < 128 * T::UPR; u += 256) {
    const int r = u / T::UPR, c = u % T::UPR;
    int i, g;
    rm.at(r, &i, &g);
    if (i < count)
      *(uint4*)(yb + ((long long)i * a.Hq + hk * G + g) * D + 8 * c) = *(const uint4*)((r < 64 ? k0 : v0) + T::at(r & 63, c));
  }
  if (__syncthreads_or(redo != 0) && redo) chunk_redo<bf16, D, BK, 32>(redo);
}

template <int D, bool SMALL> __global__ void __launch_bounds__(256, 2) chunk_bf16_kernel(ChunkAttnArgs a) {
  constexpr int BYTES = 64 * Tile<D>::RB;
  // two buffers of K and V, each a variable of its own: what is read from one
  // then does not wait for the loads into the other
  __shared__ __attribute__((aligned(16))) char k0[BYTES], v0[BYTES], k1[BYTES], v1[BYTES];
  __shared__ ChunkShortShared<bf16> sh;
  const int n_long = a.items * a.parts * a.Hkv;
  if ((int)blockIdx.x < n_long) chunk_long<D, SMALL>(a, k0, v0, k1, v1);
  else chunk_short<bf16, D>(a, blockIdx.x - n_long, [&](int v) { return v == 0 ? k0 : v == 1 ? v0 : v == 2 ? k1 : v1; }, sh);
}

template <int D> static void launch(const ChunkAttnArgs& a, unsigned groups, hipStream_t stream) {
  if (1 << a.page_log < PagedTileLoad<D, false>::ROWS)
    hipLaunchKernelGGL((chunk_bf16_kernel<D, true>), dim3(groups), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((chunk_bf16_kernel<D, false>), dim3(groups), dim3(256), 0, stream, a);
}

int chunk_bf16_launch(const ChunkAttnArgs& a, unsigned groups, hipStream_t stream) {
  if (a.D == 128) launch<128>(a, groups, stream);
  else launch<64>(a, groups, stream);
  return check_launch("chunk_bf16_kernel");
}

}  // namespace gdnx
