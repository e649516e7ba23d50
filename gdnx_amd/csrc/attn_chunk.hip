// Attention of packed new tokens over a paged key-value cache (gfx950):
// prompts' pieces, drafts and single tokens in one call.
//
// Row i's n new tokens stand at the last n positions of its table row (its
// length counts them, and their keys and values are in their pages); the one
// at p sees key j if j <= p and p - j < window or j < sinks.  A key without a
// page is not seen.
//
// The form here is the plain one: a wave takes a query head of a token, 64 keys
// at a time, a lane a key for the scores and D / 64 columns for the sum.
#include "attn_common.hpp"
#include "packed_rows.hpp"

namespace gdnx {

namespace {

// A query from what it sees alone.
template <typename CT, int D> struct ChunkRow {
  static constexpr int E = D / 64;
  float m, l, acc[E];
  __device__ __forceinline__ ChunkRow(const ChunkAttnArgs& a, const CT* q, int r, int hk, int p, int len, int lane)
      : m(-INFINITY), l(0.f) {
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    const int* table = a.table + (long long)r * a.width;
    const int mask = (1 << a.page_log) - 1;
    const KeyTiles<64> kt(p, p, len, a.window, a.sinks);
    for (int it = 0; it < kt.count; ++it) {
      const int j = kt.start(it) + lane;
      const int pg = attn_visible(p, j, a.window, a.sinks) ? table[j >> a.page_log] : -1;
      const bool vis = pg >= 0 && pg < a.n_pages;
      const long long at = vis ? (((long long)pg * a.Hkv + hk) << a.page_log) + (j & mask) : 0;     // its row in the pool
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
  }
};

}  // namespace

template <typename CT, int D> __global__ void __launch_bounds__(256) chunk_attn_kernel(ChunkAttnArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long long u = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = (int)(u % a.Hq), t = (int)(u / a.Hq);
  if (t >= a.N) return;
  const int i = wave_find(a.n, t, lane, [&](int i) { return (long long)packed_offset(a.offsets, i, a.N); });
  if (i < 0) return;
  const int first = packed_offset(a.offsets, i, a.N), count = packed_offset(a.offsets, i + 1, a.N) - first;
  if (t - first >= count) return;                  // behind the last row
  const int r = a.slots ? a.slots[i] : i;
  const long long cap = (long long)a.width << a.page_log;
  int len = r >= 0 && r < a.rows ? a.lengths[r] : 0;
  len = len < 0 || len > cap ? 0 : len;
  const int p = len - count + t - first;
  CT* y = (CT*)a.y + ((long long)t * a.Hq + h) * D + lane * E;
  if (len == 0 || p < 0) {
    for (int e = 0; e < E; ++e) y[e] = from_f<CT>(0.f);
    return;
  }
  const ChunkRow<CT, D> c(a, (const CT*)a.q + t * a.qs[0] + h * a.qs[1], r, h / (a.Hq / a.Hkv), p, len, lane);
  const float inv = c.l == 0.f ? 0.f : 1.f / c.l;
  for (int e = 0; e < E; ++e) y[e] = from_f<CT>(c.acc[e] * inv);
}

template <typename CT, int D> static int launch(const ChunkAttnArgs& a, hipStream_t stream) {
  const long long groups = ((long long)a.N * a.Hq + 3) / 4;
  hipLaunchKernelGGL((chunk_attn_kernel<CT, D>), dim3((unsigned)groups), dim3(256), 0, stream, a);
  return check_launch("chunk_attn_kernel");
}

int chunk_attn_dispatch(const ChunkAttnArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16) return a.D == 128 ? launch<bf16, 128>(a, stream) : launch<bf16, 64>(a, stream);
  return a.D == 128 ? launch<float, 128>(a, stream) : launch<float, 64>(a, stream);
}

}  // namespace gdnx
