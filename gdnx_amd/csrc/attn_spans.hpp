// Work shared out over a long axis, and its parts joined in order: the
// forward's and dq's keys where rows are few, the dk / dv kernel's rows where a key
// tile is seen by many (sinks, no window).
#pragma once
#include "attn_common.hpp"

namespace gdnx {

// ---- forward: rows that are gone over again ----
// In a tile that a row sees in part, a hidden value enters its product times
// zero, which is NaN where the value is not finite.  So a row whose output is
// not finite is formed again, by its whole wave, from what it sees alone: 64
// keys at a time, a lane a key for the scores and D / 64 columns for the sum.
// Nothing of this runs while all outputs are finite.
template <typename CT, int D, int BK> struct CarefulRow {
  static constexpr int E = D / 64;
  float m, l, acc[E];
  __device__ __forceinline__ CarefulRow(const WinAttnArgs& a, const CT* q, const CT* kb, const CT* vb,
                                        const KeyTiles<BK>& kt, int t0, int t1, int p, int lane)
      : m(-INFINITY), l(0.f) {
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int it = t0; it < t1; ++it)
      for (int jb = kt.start(it); jb < kt.start(it) + BK; jb += 64) {
        const int j = jb + lane;
        const bool vis = lane < BK && attn_visible(p, j, a.window, a.sinks);
        float s = 0.f;
        if (vis)
          for (int d = 0; d < D; ++d) s = fmaf(to_f(q[d]), to_f(kb[j * a.ks[1] + d]), s);
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
          for (int e = 0; e < E; ++e) acc[e] = fmaf(pk, to_f(vb[(jb + key) * a.vs[1] + lane * E + e]), acc[e]);
        }
      }
  }
};

// ---- forward: parts of a row's keys ----
__device__ __forceinline__ float* part_out(const WinAttnArgs& a, int part, long long row) {
  return a.part + ((long long)part * a.B * a.Hq * a.Tq + row) * a.D;
}
__device__ __forceinline__ float* part_stats(const WinAttnArgs& a, int part, long long row) {
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  return a.part + (long long)a.parts * rows * a.D + 2 * (part * rows + row);
}

// D / 4 threads a row ([B,Tq,Hq]), four columns each.
template <typename CT, int D> __global__ void __launch_bounds__(256) win_join_kernel(WinAttnArgs a) {
  constexpr int V = D / 4;
  const long long rows = (long long)a.B * a.Hq * a.Tq, r = (long long)blockIdx.x * (256 / V) + threadIdx.x / V;
  if (r >= rows) return;
  const int d = 4 * (threadIdx.x % V);
  float m = -INFINITY, l = 0.f;
  f32x4 acc = zero4();
#pragma unroll 4
  for (int i = 0; i < a.parts; ++i) {
    const float* ml = part_stats(a, i, r);
    const f32x4 x = *(const f32x4*)(part_out(a, i, r) + d);
    const float mn = fmaxf(m, ml[0]), ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ms), g = __builtin_amdgcn_exp2f(ml[0] - ms);
    l = l * f + ml[1] * g;
    acc = acc * f + x * g;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  acc *= inv;
  st4((CT*)a.y + r * D + d, acc[0], acc[1], acc[2], acc[3]);
  if (a.y_low)
    st4((CT*)a.y_low + r * D + d, bf16_rest(acc[0]), bf16_rest(acc[1]), bf16_rest(acc[2]), bf16_rest(acc[3]));
  if (d == 0 && a.lse) {
    const int h = (int)(r % a.Hq);
    const long long bi = r / a.Hq;
    a.lse[((bi / a.Tq) * a.Hq + h) * a.Tq + bi % a.Tq] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
  }
}

// The rows of the wave in `redo` (a bit for each of its WR rows) formed again
// and stored over what the workgroup has stored before its last barrier.  All
// of it is read and worked out anew from the kernel's arguments, the first
// and only ones of a forward kernel of 4 WR rows a workgroup: held from the
// kernel's start, it took registers from the main loop (5 % of its time).
template <typename CT, int D, int BK, int WR> __device__ __forceinline__ void careful_rows(unsigned redo) {
  constexpr int E = D / 64;
  const auto* args = (const __attribute__((address_space(4))) WinAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  int w = blockIdx.x, tid = opaque(threadIdx.x);
  asm volatile("" : "+s"(args), "+s"(w));
  WinAttnArgs a;
  __builtin_memcpy(&a, (const void*)args, sizeof(a));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, nt = (a.Tq * G + 4 * WR - 1) / (4 * WR), off = a.Tk - a.Tq;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int part = w % a.parts, tile = nt - 1 - w / a.parts;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  const RowMap rm(tile * 4 * WR, G, a.g_magic);
  const KeyTiles<BK> kt(rm.i0 + off, min(rm.last(4 * WR - 1), a.Tq - 1) + off, len, a.window, a.sinks);
  const int per = (kt.count + a.parts - 1) / a.parts, t0 = part * per, t1 = min(kt.count, t0 + per);
  const CT* kb = (const CT*)a.k + b * a.ks[0] + hk * a.ks[2];
  const CT* vb = (const CT*)a.v + b * a.vs[0] + hk * a.vs[2];
  for (; redo; redo &= redo - 1) {
    int i, h;
    rm.at(wave * WR + __ffs(redo) - 1, &i, &h);
    h += hk * G;
    const CT* q = (const CT*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
    const CarefulRow<CT, D, BK> c(a, q, kb, vb, kt, t0, t1, i + off, lane);
    const long long r = ((long long)b * a.Tq + i) * a.Hq + h;
    const float inv = c.l == 0.f ? 0.f : 1.f / c.l;
    for (int e = 0; e < E; ++e) {
      if (a.parts > 1) {
        part_out(a, part, r)[lane * E + e] = c.acc[e];
        continue;
      }
      ((CT*)a.y)[r * D + lane * E + e] = from_f<CT>(c.acc[e] * inv);
      if (a.y_low) ((CT*)a.y_low)[r * D + lane * E + e] = from_f<CT>(bf16_rest(c.acc[e] * inv));
    }
    if (lane == 0) {
      if (a.parts > 1) {
        part_stats(a, part, r)[0] = c.m;
        part_stats(a, part, r)[1] = c.l;
      } else if (a.lse) {
        a.lse[((long long)b * a.Hq + h) * a.Tq + i] = c.l == 0.f ? -INFINITY : c.m * kLn2 + logf(c.l);
      }
    }
  }
}

template <typename CT, int D> static int launch_win_join(const WinAttnArgs& a, hipStream_t stream) {
  if (a.parts == 1) return GDNX_OK;
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  hipLaunchKernelGGL((win_join_kernel<CT, D>), dim3((unsigned)((rows + 1024 / D - 1) / (1024 / D))), dim3(256), 0, stream,
                     a);
  return check_launch("win_join_kernel");
}

// ---- dq: parts of a row's keys, [parts][B,Tq,Hq,D] ----
template <typename CT> __global__ void __launch_bounds__(256) win_dq_join_kernel(WinAttnBwdArgs a) {
  const long long n = (long long)a.B * a.Tq * a.Hq * a.D, u = 4 * ((long long)blockIdx.x * 256 + threadIdx.x);
  if (u >= n) return;
  f32x4 x = zero4();
  for (int p = 0; p < a.dq_parts; ++p) x += *(const f32x4*)(a.part + p * n + u);
  x *= a.scale;
  st4((CT*)a.dq + u, x[0], x[1], x[2], x[3]);
}

template <typename CT> static int launch_dq_join(const WinAttnBwdArgs& a, hipStream_t stream) {
  if (a.dq_parts == 1) return GDNX_OK;
  const long long n = (long long)a.B * a.Tq * a.Hq * a.D;
  hipLaunchKernelGGL((win_dq_join_kernel<CT>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream, a);
  return check_launch("win_dq_join_kernel");
}

// ---- dk, dv: spans of a key tile's rows ----
// The 64-row steps that the KT keys from k0 take, cut into as few parts as
// hold a.span steps at most, of one size (`per`).
template <int KT> struct KeySpan {
  int i0;              // the first query
  int rows;            // rows (query, head) from there on
  int steps, parts, per;
  __device__ __forceinline__ KeySpan(const WinAttnBwdArgs& a, int k0, int len) {
    const int off = a.Tk - a.Tq, p0 = max(k0, off), pe = k0 < len ? last_query<KT>(k0, len, a.window, a.sinks) : 0;
    i0 = p0 - off;
    rows = pe > p0 ? (pe - p0) * (a.Hq / a.Hkv) : 0;
    steps = (rows + 63) / 64;
    parts = max(1, (steps + a.span - 1) / a.span);
    per = (steps + parts - 1) / parts;
  }
};

// A head's slots: the tiles that hold sinks first, each with its most parts.
template <int KT> __host__ __device__ __forceinline__ long long span_slots(const WinAttnBwdArgs& a) {
  return (long long)a.sink_tiles * a.sink_parts + ((long long)(a.Tk + KT - 1) / KT - a.sink_tiles) * a.tile_parts;
}
struct SpanSlot {
  int tile, part;
  __device__ __forceinline__ SpanSlot(const WinAttnBwdArgs& a, int w) {
    const int n = a.sink_tiles * a.sink_parts;
    tile = w < n ? w / a.sink_parts : a.sink_tiles + (w - n) / a.tile_parts;
    part = w < n ? w % a.sink_parts : (w - n) % a.tile_parts;
  }
};

// A key tile's parts summed in order, four columns of dk or dv a thread.
template <typename CT, int D, int KT> __global__ void __launch_bounds__(256) win_dkv_join_kernel(WinAttnBwdArgs a) {
  constexpr int BLK = 2 * KT * D / 1024;             // workgroups a tile
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int kt = w / BLK, u = 4 * ((w % BLK) * 256 + threadIdx.x);   // of [dk, dv][KT][D]
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  const KeySpan<KT> ks(a, kt * KT, len);
  const int key = kt * KT + u / D % KT, d = u % D;
  if (ks.parts <= 1 || key >= a.Tk) return;
  const int first = kt < a.sink_tiles ? kt * a.sink_parts : a.sink_tiles * a.sink_parts + (kt - a.sink_tiles) * a.tile_parts;
  const float* part = a.part + (((long long)b * a.Hkv + hk) * span_slots<KT>(a) + first) * 2 * KT * D + u;
  f32x4 x = zero4();
#pragma unroll 4
  for (int p = 0; p < ks.parts; ++p) x += *(const f32x4*)(part + (long long)p * 2 * KT * D);
  const bool dk = u < KT * D;
  if (dk) x *= a.scale;
  st4((CT*)(dk ? a.dk : a.dv) + (((long long)b * a.Tk + key) * a.Hkv + hk) * D + d, x[0], x[1], x[2], x[3]);
}

template <typename CT, int D, int KT> static int launch_dkv_join(const WinAttnBwdArgs& a, hipStream_t stream) {
  if (a.tile_parts == 1 && (a.sink_tiles == 0 || a.sink_parts == 1)) return GDNX_OK;
  // (with a window often only the tiles with sinks have several parts)
  const long long tiles = a.tile_parts > 1 ? (a.Tk + KT - 1) / KT : a.sink_tiles;
  hipLaunchKernelGGL((win_dkv_join_kernel<CT, D, KT>), dim3((unsigned)(tiles * (2 * KT * D / 1024) * a.B * a.Hkv)), dim3(256), 0,
                     stream, a);
  return check_launch("win_dkv_join_kernel");
}

}  // namespace gdnx
