// Work shared out over a long axis, and its parts joined in order: the
// forward's and dq's keys where rows are few, the dk / dv kernel's rows where a key
// tile is seen by many (sinks, no window).
#pragma once
#include "attn_common.hpp"

namespace gdnx {

// ---- forward: parts of a row's keys ----
__device__ __forceinline__ float* part_out(const WinAttnArgs& a, int part, long long row) {
  return a.part + ((long long)part * a.B * a.Hq * a.Tq + row) * a.D;
}
__device__ __forceinline__ float* part_stats(const WinAttnArgs& a, int part, long long row) {
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  return a.part + (long long)a.parts * rows * a.D + 2 * (part * rows + row);
}

// One wave a row ([B,Tq,Hq]).
template <typename CT, int D> __global__ void __launch_bounds__(256) win_join_kernel(WinAttnArgs a) {
  constexpr int E = D / 64;
  const long long rows = (long long)a.B * a.Hq * a.Tq, r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int lane = threadIdx.x & 63;
  float mm = -INFINITY;
  for (int i = 0; i < a.parts; ++i) mm = fmaxf(mm, part_stats(a, i, r)[0]);
  const float ms = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int i = 0; i < a.parts; ++i) {
    const float f = __builtin_amdgcn_exp2f(part_stats(a, i, r)[0] - ms);
    ll += part_stats(a, i, r)[1] * f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += part_out(a, i, r)[lane * E + e] * f;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    ((CT*)a.y)[r * D + lane * E + e] = from_f<CT>(acc[e] * inv);
    if (a.y_low) ((CT*)a.y_low)[r * D + lane * E + e] = from_f<CT>(bf16_rest(acc[e] * inv));
  }
  if (lane == 0 && a.lse) {
    const int h = (int)(r % a.Hq);
    const long long bi = r / a.Hq;
    a.lse[((bi / a.Tq) * a.Hq + h) * a.Tq + bi % a.Tq] = ll == 0.f ? -INFINITY : mm * kLn2 + logf(ll);
  }
}

template <typename CT, int D> static int launch_win_join(const WinAttnArgs& a, hipStream_t stream) {
  if (a.parts == 1) return GDNX_OK;
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  hipLaunchKernelGGL((win_join_kernel<CT, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
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

// 32 keys a workgroup: their parts summed in order.
template <typename CT, int D, int KT> __global__ void __launch_bounds__(256) win_dkv_join_kernel(WinAttnBwdArgs a) {
  constexpr int V = D / 4, RPW = 256 / V, BLK = KT / 32;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int blk = w % BLK, kt = w / BLK;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  const KeySpan<KT> ks(a, kt * KT, len);
  if (ks.parts <= 1) return;
  const int first = kt < a.sink_tiles ? kt * a.sink_parts : a.sink_tiles * a.sink_parts + (kt - a.sink_tiles) * a.tile_parts;
  const long long slot = ((long long)b * a.Hkv + hk) * span_slots<KT>(a) + first;
  const int d = 4 * (threadIdx.x % V);
  for (int r = blk * 32 + threadIdx.x / V; r < blk * 32 + 32; r += RPW) {
    if (kt * KT + r >= a.Tk) break;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f32x4 x = zero4();
      for (int p = 0; p < ks.parts; ++p) x += *(const f32x4*)(a.part + ((slot + p) * 2 * KT + m * KT + r) * D + d);
      if (m == 0) x *= a.scale;
      st4((CT*)(m ? a.dv : a.dk) + (((long long)b * a.Tk + kt * KT + r) * a.Hkv + hk) * D + d, x[0], x[1], x[2], x[3]);
    }
  }
}

template <typename CT, int D, int KT> static int launch_dkv_join(const WinAttnBwdArgs& a, hipStream_t stream) {
  if (a.tile_parts == 1 && (a.sink_tiles == 0 || a.sink_parts == 1)) return GDNX_OK;
  // (with a window often only the tiles with sinks have several parts)
  const long long tiles = a.tile_parts > 1 ? (a.Tk + KT - 1) / KT : a.sink_tiles;
  hipLaunchKernelGGL((win_dkv_join_kernel<CT, D, KT>), dim3((unsigned)(tiles * (KT / 32) * a.B * a.Hkv)), dim3(256), 0,
                     stream, a);
  return check_launch("win_dkv_join_kernel");
}

}  // namespace gdnx
