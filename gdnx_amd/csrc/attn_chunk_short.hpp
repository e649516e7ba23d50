// Short rows of a packed batch (single tokens, drafts): at most 32 (16 in
// float32, whose registers do not hold more: 64 rows of up to 4000 tokens, d = 128,
// 238 us with 32, 118 with 16) (token, query head of the group) pairs of one key head, whose keys a workgroup's four
// waves take in turn, a tile of 32 (16 in float32) each, straight to registers
// as the served step does (attn_paged.hip): bound by memory, each visible key and
// value is read once for all pairs.  Spans of long rows are joined by a second
// kernel, in order.  Few rows wait for one lookup after the other (offsets and
// slot, length, page, keys), so queries are asked for after the first page and masks
// are formed where a tile needs them: 8 rows of 5 tokens on up to 2000, 16/4 heads,
// 13.3 us (16.2 with every tile masked and rescaled, and the waves' join by
// straight rows in LDS).
#pragma once
#include "attn_chunk.hpp"
#include "attn_paged.hpp"

namespace gdnx {

template <typename CT> struct ChunkShortShared {
  static constexpr int BT = FragT<CT>::KSTEP;
  long long off[4][BT];
  float m[4][kChunkShort], l[4][kChunkShort];
  unsigned bad;
};

// buf(v): LDS of wave v, 32 D floats.
template <typename CT, int D, typename Buf>
__device__ __forceinline__ void chunk_short(const ChunkAttnArgs& a, int w, const Buf& buf, ChunkShortShared<CT>& sh) {
  typedef typename FragT<CT>::type Frag;
  constexpr int BT = FragT<CT>::KSTEP, NU = FragT<CT>::TPS, NB = chunk_short_pairs(sizeof(CT)) / 16;
  constexpr int EPU = 16 / sizeof(CT), UPR = D / EPU, NKS = D / FragT<CT>::KSTEP, NT = D / 16;
  constexpr int NV = BT * UPR / 64;                               // 16-byte units of a V tile a lane
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.Hq / a.Hkv;
  const int span = w % a.spans; w /= a.spans;
  const int hk = w % a.Hkv, i = w / a.Hkv;
  const int first = packed_offset(a.offsets, i, a.N), count = packed_offset(a.offsets, i + 1, a.N) - first;
  ChunkSeq s;                                                     // (looked up beside the offsets, not after them)
  s.find(a, i, first, count);
  if (count <= 0 || (long long)count * G > a.short_rows) return;
  const ChunkSeen see(a, s);
  const int rows = count * G, blocks = (rows + 15) / 16;
  const int tiles = (see.nvis + BT - 1) / BT, parts = chunk_spans(tiles, a.spans);
  const RowMap rm(0, G, a.g_magic);
  // the pair of row q: its place in q and y
  const auto pair_at = [&](int q, int* qi, int* h) {
    rm.at(q, qi, h);
    *h += hk * G;
  };
  if (span >= parts) {
    if (span == 0)                                                // an empty row
      for (int u = tid; u < rows * (D / 4); u += 256) {
        int qi, h;
        pair_at(u / (D / 4), &qi, &h);
        st4((CT*)a.y + ((long long)(first + qi) * a.Hq + h) * D + 4 * (u % (D / 4)), 0.f, 0.f, 0.f, 0.f);
      }
    return;
  }
  const int* table = a.table + (long long)s.r * a.width;
  const long long rowb = D * (int)sizeof(CT), headb = rowb << a.page_log;
  const int per = (tiles + parts - 1) / parts, t0 = span * per, t1 = min(tiles, t0 + per);

  const auto page_of = [&](int x) { return x < see.nvis ? table[see.key(x) >> a.page_log] : -1; };
  int t = t0 + wave;
  int pg = t < t1 && lane < BT ? page_of(t * BT + lane) : -1;
  Frag qf[NB][NKS];
  int pos[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    int qi, h;
    pair_at(16 * b + n, &qi, &h);
    const bool there = 16 * b + n < rows;
    pos[b] = there ? s.off + qi : -1;
#pragma unroll
    for (int c = 0; c < NKS; ++c) {
      if (there) qf[b][c] = *(const Frag*)((const CT*)a.q + (first + qi) * a.qs[0] + h * a.qs[1] + (4 * c + g) * EPU);
      else qf[b][c] = Frag{};
      if (a.scale < 0.f) qf[b][c] = -qf[b][c];
    }
  }
  Frag kr[NU][NKS];
  u32x4 vr[NV];
  bool live[NU];                       // whether the lane's keys of the tile are there
  long long* off = sh.off[wave];
  CT* stage = (CT*)buf(wave);
  const auto load = [&](int t, int pg) {
    wave_lds_sync();
    if (lane < BT) {
      const int x = t * BT + lane;
      off[lane] = x < see.nvis && pg >= 0 && pg < a.n_pages
                      ? ((long long)pg * a.Hkv + hk) * headb + (see.key(x) & ((1 << a.page_log) - 1)) * rowb : -1;
    }
    wave_lds_sync();
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const long long o = off[16 * u + n];
      const GlobalBytes p = (GlobalBytes)(o >= 0 ? (const char*)a.k_pages + o : (const char*)g_zero_row);
      live[u] = o >= 0;
#pragma unroll
      for (int c = 0; c < NKS; ++c) kr[u][c] = ld_global<Frag>(p + (4 * c + g) * 16);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int U = i * 64 + lane, row = U / UPR, u = (U % UPR) ^ v_swizzle<D>((const CT*)nullptr, row);
      const long long o = off[row];
      const GlobalBytes p = (GlobalBytes)(o >= 0 ? (const char*)a.v_pages + o : (const char*)g_zero_row);
      vr[i] = ld_global<u32x4>(p + u * 16);
    }
  };

  const float size = fabsf(a.scale) * kLog2e, sc = size < 1e-30f ? 1e-30f : size;      // (no number stays none)
  f32x4 o[NB][NT];
  float m[NB], l[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int t = 0; t < NT; ++t) o[b][t] = zero4();
    m[b] = -INFINITY;
    l[b] = 0.f;
  }
  if (t < t1) load(t, pg);
  pg = t + 4 < t1 && lane < BT ? page_of((t + 4) * BT + lane) : -1;
  for (; t < t1; t += 4) {
    f32x4 sx[NB][NU];
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (b < blocks) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          sx[b][u] = zero4();
#pragma unroll
          for (int c = 0; c < NKS; ++c) mma(sx[b][u], kr[u][c], qf[b][c]);
        }
      }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < NV; ++i) *(u32x4*)((char*)stage + (i * 64 + lane) * 16) = vr[i];
    // whether all the tokens see all of the tile (a single one what is there); else which keys of the lane's
    // accumulator rows are seen: lane 4 g + e has key 16 u + 4 g + e
    const int k0 = see.key(t * BT), k1 = see.key(t * BT + BT - 1);
    bool all = count == 1 || (k1 <= s.off && (s.off + count - 1 - k0 < a.window || k1 < a.sinks));
#pragma unroll
    for (int u = 0; u < NU; ++u) all = all && __all(live[u]);
    if (!all) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const unsigned long long lv = __ballot(live[u]) >> (4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = see.key(t * BT + 16 * u + 4 * g + e);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            if (b < blocks)
              sx[b][u][e] = (lv >> e & 1) && (count == 1 || attn_visible(pos[b], j, a.window, a.sinks)) ? sx[b][u][e] : -INFINITY;
        }
      }
    }
    if (t + 4 < t1) {
      load(t + 4, pg);
      pg = t + 8 < t1 && lane < BT ? page_of((t + 8) * BT + lane) : -1;
    }
    Frag pf[NB], pr[NB];                 // P, and what rounding it to bf16 leaves over
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (b < blocks) {
        float mx = sx[b][0][0];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sx[b][u][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * sc;
        if (__any(mx > m[b] + 8.f)) {        // (raised by steps of 2^8)
          const float mn = fmaxf(m[b], mx), f = __builtin_amdgcn_exp2f(m[b] - (mn == -INFINITY ? 0.f : mn));
          m[b] = mn;
          l[b] *= f;
#pragma unroll
          for (int c = 0; c < NT; ++c) o[b][c] *= f;
        }
        const float ms = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sx[b][u][e] = __builtin_amdgcn_exp2f(fmaf(sx[b][u][e], sc, -ms));
            l[b] += sx[b][u][e];
          }
        pf[b] = acc_frag((CT*)nullptr, sx[b][0], sx[b][NU - 1]);
        if constexpr (sizeof(CT) == 2) {
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sx[b][u][e] = bf16_rest(sx[b][u][e]);
          pr[b] = acc_frag((CT*)nullptr, sx[b][0], sx[b][NU - 1]);
        }
      }
    wave_lds_sync();
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const Frag vf = v_frag<D>(stage, c, n, g);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (b < blocks) {
          mma(o[b][c], vf, pf[b]);
          if constexpr (sizeof(CT) == 2) mma(o[b][c], vf, pr[b]);
        }
    }
  }
  // the four waves joined
  if (tid == 0) sh.bad = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (b < blocks) {
      l[b] += __shfl_xor(l[b], 16, 64);
      l[b] += __shfl_xor(l[b], 32, 64);
      if (g == 0) {
        sh.m[wave][16 * b + n] = m[b];
        sh.l[wave][16 * b + n] = l[b];
      }
    }
  wave_lds_sync();
  float* so = (float*)buf(wave);         // a row's 16-byte units by an xor, so that 16 rows are stored without a bank conflict
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (b < blocks) {
#pragma unroll
      for (int c = 0; c < NT; ++c) *(f32x4*)&so[(16 * b + n) * D + 4 * ((4 * c + g) ^ n)] = o[b][c];
    }
  __syncthreads();
  for (int u = tid; u < rows * (D / 4); u += 256) {
    const int q = u / (D / 4), d = 4 * (u % (D / 4));
    float mm = sh.m[0][q];
#pragma unroll
    for (int v = 1; v < 4; ++v) mm = fmaxf(mm, sh.m[v][q]);
    const float ms = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    f32x4 acc = zero4();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = __builtin_amdgcn_exp2f(sh.m[v][q] - ms);
      ll += sh.l[v][q] * f;
      acc += *(const f32x4*)&((const float*)buf(v))[q * D + (d ^ 4 * (q & 15))] * f;
    }
    if (fmaf(acc[0], 0.f, fmaf(acc[1], 0.f, fmaf(acc[2], 0.f, acc[3] * 0.f))) != 0.f) atomicOr(&sh.bad, 1u << q);
    int qi, h;
    pair_at(q, &qi, &h);
    if (parts == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      st4((CT*)a.y + ((long long)(first + qi) * a.Hq + h) * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      const long long row = ((long long)i * a.Hkv + hk) * kChunkShort + q;
      *(f32x4*)(short_out(a, row, span) + d) = acc;
      if (d == 0) {
        float* ml = short_stats(a, row, span);
        ml[0] = mm;
        ml[1] = ll;
      }
    }
  }
  __syncthreads();
  const int x1 = min(see.nvis, t1 * BT);
  for (unsigned redo = sh.bad; redo; redo &= redo - 1) {          // rows whose output is not finite
    const int q = __ffs(redo) - 1;
    if ((q & 3) != wave) continue;
    int qi, h;
    pair_at(q, &qi, &h);
    const CT* qp = (const CT*)a.q + (first + qi) * a.qs[0] + h * a.qs[1];
    ChunkRow<CT, D> c;
    for (int x = t0 * BT; x < x1; x += 64) c.add(a, qp, s.r, hk, s.off + qi, x + lane < x1 ? see.key(x + lane) : -1, lane);
    const long long row = ((long long)i * a.Hkv + hk) * kChunkShort + q;
    if (parts == 1) c.store((CT*)a.y + ((long long)(first + qi) * a.Hq + h) * D, lane);
    else c.store_part(short_out(a, row, span), short_stats(a, row, span), lane);
  }
}

}  // namespace gdnx
