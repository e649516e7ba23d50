// Attention with a sliding window and sinks (gfx950): the rules, the shares of
// the work, and the float32 kernels.
//
//   P_ij = exp(s q_i.k_j - lse_i) over the visible j,  y_i = sum_j P_ij v_j
//   dV = P^T dY;  dP = dY V^T;  dS = P o (dP - delta),  delta_i = dY_i.Y_i;
//   dQ = s dS K;  dK = s dS^T Q, both summed over a key head's query heads.
//
// Rows are (query, query head of the group) pairs with the heads fastest, so
// grouped heads share the key tiles and a tile's rows span few positions.  The
// scores are formed transposed to what they are contracted over next, so that
// a score tile's accumulators are the next product's operand: S^T = K Q^T
// feeds O^T = V^T P^T and dQ^T = K^T dS^T; S = Q K^T feeds dV^T = dY^T P and
// dK^T = Q^T dS.  Softmax statistics, sums and products are float32.
//
// Float32: v_mfma_f32_16x16x4_f32, a wave owns 16 rows (forward, dq) or 16
// keys (dk, dv); tiles of 32 keys (rows) by way of registers into LDS,
// double-buffered, one barrier a tile.  Rows of a tile are D + 4 words apart,
// which keeps both reads (16 rows of 4 words, 4 x 16 words) off each other's
// banks.  Bound by the matrix units, which the forward keeps busy 59 % of the
// cycles, dq 67 %, dk / dv 50 %: B = 2, T = 4096, 8/4 heads, d = 128, window
// 512 take 190 us forward (86 TFLOP/s) and 695 us backward (58; a float32
// library product of size 8192 reaches 154).
#include "attn_f32.hpp"
#include "attn_spans.hpp"

namespace gdnx {

namespace {

// The rows of a workgroup of the forward and dq: 64 rows, a lane's row n of
// its wave's 16, and the positions that they span.
struct F32Rows {
  RowMap rm;
  int i, h, p, wg0, wg1, wv0, wv1;
  bool rows_ok;
  __device__ __forceinline__ F32Rows(int tile, int wave, int n, int hk, int G, unsigned magic, int Tq, int off, int len)
      : rm(tile * 64, G, magic) {
    rm.at(wave * 16 + n, &i, &h);
    h += hk * G;
    p = i < Tq && i + off < len ? i + off : -1;
    wg0 = rm.i0 + off;
    wg1 = min(rm.last(63), Tq - 1) + off;
    wv0 = rm.last(wave * 16) + off;
    const int last = rm.last(wave * 16 + 15);
    wv1 = min(min(last, Tq - 1) + off, len - 1);
    rows_ok = last < Tq && last + off < len && wv0 >= 0;
  }
  __device__ __forceinline__ bool some(int j0, int window, int sinks) const {
    return wv0 <= wv1 && j0 <= wv1 && (j0 + 31 > wv0 - window || j0 < sinks);
  }
  __device__ __forceinline__ bool all(int j0, int window, int sinks) const {
    return rows_ok && j0 + 31 <= wv0 && (wv1 - j0 < window || j0 + 32 <= sinks);
  }
};

}  // namespace

template <int D> __global__ void __launch_bounds__(256, 2) win_fwd_f32_kernel(WinAttnArgs a) {
  using T = F32Tile<D>;
  __shared__ __attribute__((aligned(16))) float smem[4 * T::WORDS];       // two buffers of K, V
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, nt = (a.Tq * G + 63) / 64;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int part = w % a.parts, tile = nt - 1 - w / a.parts;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const F32Rows rows(tile, wave, n, hk, G, a.g_magic, a.Tq, off, len);
  const float* kb = (const float*)a.k + b * a.ks[0] + hk * a.ks[2];
  const float* vb = (const float*)a.v + b * a.vs[0] + hk * a.vs[2];
  f32x4 qf[T::NS];
  {
    const float* qp = (const float*)a.q + b * a.qs[0] + (rows.p >= 0 ? rows.i * a.qs[1] + rows.h * a.qs[2] : 0);
#pragma unroll
    for (int c = 0; c < T::NS; ++c) qf[c] = *(const f32x4*)(qp + 16 * c + 4 * g);
  }
  const float sc = a.scale * kLog2e;
  const KeyTiles<32> kt(rows.wg0, rows.wg1, len, a.window, a.sinks);
  const int per = (kt.count + a.parts - 1) / a.parts, t0 = part * per, t1 = min(kt.count, t0 + per);
  F32Stage<D> st(tid);
  const auto load = [&](int it) {
    const int j0 = kt.start(it);
    st.load([&](int r, const float** x, const float** y) {
      const long long j = min(j0 + r, len - 1);
      *x = kb + j * a.ks[1];
      *y = vb + j * a.vs[1];
    });
  };
  f32x4 o[T::NS];
#pragma unroll
  for (int t = 0; t < T::NS; ++t) o[t] = zero4();
  float m = -INFINITY, l = 0.f;
  if (t0 < t1) {
    load(t0);
    st.store(smem, smem + T::WORDS);
  }
  lds_barrier();
  for (int it = t0; it < t1; ++it) {
    const int j0 = kt.start(it);
    const float *sk = smem + ((it - t0) & 1) * 2 * T::WORDS, *sv = sk + T::WORDS;
    load(min(it + 1, t1 - 1));
    if (rows.some(j0, a.window, a.sinks)) {
      const bool all = rows.all(j0, a.window, a.sinks);
      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = zero4();
#pragma unroll
        for (int c = 0; c < T::NS; ++c) mma(s[u], ld_frag(sk + (16 * u + n) * T::LD + 16 * c, g), qf[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[u][e] = all || attn_visible(rows.p, j0 + 16 * u + 4 * g + e, a.window, a.sinks) ? s[u][e] * sc : -INFINITY;
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m - ms);
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][e] = exp2f(s[u][e] - ms);
          sum += s[u][e];
        }
      l = l * f + sum;
      m = mn;
#pragma unroll
      for (int t = 0; t < T::NS; ++t) {
        o[t] *= f;
#pragma unroll
        for (int u = 0; u < 2; ++u) mma(o[t], ld_cols<T::LD>(sv, 16 * u, 16 * t + n, g), s[u]);
      }
    }
    float* next = smem + ((it - t0 + 1) & 1) * 2 * T::WORDS;
    st.store(next, next + T::WORDS);
    lds_barrier();
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (rows.p < 0) {                         // a row that sees nothing: 0 times a value that is not finite is NaN
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
  const long long r = ((long long)b * a.Tq + rows.i) * a.Hq + rows.h;
  if (rows.i < a.Tq && a.parts > 1) {
    float* po = part_out(a, part, r) + 4 * g;
#pragma unroll
    for (int t = 0; t < T::NS; ++t) *(f32x4*)(po + 16 * t) = o[t];
    if (g == 0) {
      float* ml = part_stats(a, part, r);
      ml[0] = m;
      ml[1] = l;
    }
  } else if (rows.i < a.Tq) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < T::NS; ++t) *(f32x4*)((float*)a.y + r * D + 16 * t + 4 * g) = o[t] * inv;
    if (g == 0 && a.lse)
      a.lse[((long long)b * a.Hq + rows.h) * a.Tq + rows.i] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
  }
  if (redo) {
    __builtin_amdgcn_s_waitcnt(0x0070);             // (the wave's own stores come first)
    careful_rows<float, D, 32, 16>(redo);
  }
}

// dq, and delta for the dk / dv kernel
template <int D> __global__ void __launch_bounds__(256, 2) win_dq_f32_kernel(WinAttnBwdArgs a) {
  using T = F32Tile<D>;
  __shared__ __attribute__((aligned(16))) float smem[4 * T::WORDS];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, nt = (a.Tq * G + 63) / 64;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int part = w % a.dq_parts, tile = nt - 1 - w / a.dq_parts;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const F32Rows rows(tile, wave, n, hk, G, a.g_magic, a.Tq, off, len);
  const float* kb = (const float*)a.k + b * a.ks[0] + hk * a.ks[2];
  const float* vb = (const float*)a.v + b * a.vs[0] + hk * a.vs[2];
  const long long r = ((long long)b * a.Tq + rows.i) * a.Hq + rows.h;
  f32x4 qf[T::NS], gf[T::NS];
  float delta = 0.f, lse = 0.f;
  {
    const float* qp = (const float*)a.q + b * a.qs[0] + (rows.p >= 0 ? rows.i * a.qs[1] + rows.h * a.qs[2] : 0);
    const long long row = rows.p >= 0 ? r * D : 0, srow = ((long long)b * a.Hq + rows.h) * a.Tq + rows.i;
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      qf[c] = *(const f32x4*)(qp + 16 * c + 4 * g);
      gf[c] = *(const f32x4*)((const float*)a.dy + row + 16 * c + 4 * g);
      const f32x4 yf = *(const f32x4*)((const float*)a.y + row + 16 * c + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) delta += gf[c][e] * yf[e];
    }
    delta += __shfl_xor(delta, 16, 64);
    delta += __shfl_xor(delta, 32, 64);
    if (rows.p >= 0) {
      lse = a.lse[srow] * kLog2e;
      if (g == 0 && part == 0) a.delta[srow] = delta;
    }
  }
  const float sc = a.scale * kLog2e;
  const KeyTiles<32> kt(rows.wg0, rows.wg1, len, a.window, a.sinks);
  const int per = (kt.count + a.dq_parts - 1) / a.dq_parts, t0 = part * per, t1 = min(kt.count, t0 + per);
  F32Stage<D> st(tid);
  const auto load = [&](int it) {
    const int j0 = kt.start(it);
    st.load([&](int x, const float** pk, const float** pv) {
      const long long j = min(j0 + x, len - 1);
      *pk = kb + j * a.ks[1];
      *pv = vb + j * a.vs[1];
    });
  };
  f32x4 o[T::NS];
#pragma unroll
  for (int t = 0; t < T::NS; ++t) o[t] = zero4();
  if (t0 < t1) {
    load(t0);
    st.store(smem, smem + T::WORDS);
  }
  lds_barrier();
  for (int it = t0; it < t1; ++it) {
    const int j0 = kt.start(it);
    const float *sk = smem + ((it - t0) & 1) * 2 * T::WORDS, *sv = sk + T::WORDS;
    load(min(it + 1, t1 - 1));
    if (rows.some(j0, a.window, a.sinks)) {
      const bool all = rows.all(j0, a.window, a.sinks);
      f32x4 ds[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4 s = zero4(), dp = zero4();
#pragma unroll
        for (int c = 0; c < T::NS; ++c) {
          mma(s, ld_frag(sk + (16 * u + n) * T::LD + 16 * c, g), qf[c]);
          mma(dp, ld_frag(sv + (16 * u + n) * T::LD + 16 * c, g), gf[c]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          ds[u][e] = all || attn_visible(rows.p, j0 + 16 * u + 4 * g + e, a.window, a.sinks)
                         ? exp2f(s[e] * sc - lse) * (dp[e] - delta) : 0.f;
      }
#pragma unroll
      for (int t = 0; t < T::NS; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) mma(o[t], ld_cols<T::LD>(sk, 16 * u, 16 * t + n, g), ds[u]);
    }
    float* next = smem + ((it - t0 + 1) & 1) * 2 * T::WORDS;
    st.store(next, next + T::WORDS);
    lds_barrier();
  }
  if (rows.i >= a.Tq) return;
  if (rows.p < 0) {                         // a row that sees nothing: 0 times a key that is not finite is NaN
#pragma unroll
    for (int t = 0; t < T::NS; ++t) o[t] = zero4();
  }
  if (a.dq_parts > 1) {
#pragma unroll
    for (int t = 0; t < T::NS; ++t)
      *(f32x4*)(a.part + ((long long)part * a.B * a.Tq * a.Hq + r) * D + 16 * t + 4 * g) = o[t];
    return;
  }
#pragma unroll
  for (int t = 0; t < T::NS; ++t) *(f32x4*)((float*)a.dq + r * D + 16 * t + 4 * g) = o[t] * a.scale;
}

// dk, dv of 64 keys over a span of the rows that see them, 32 rows a step
template <int D> __global__ void __launch_bounds__(256, 2) win_dkv_f32_kernel(WinAttnBwdArgs a) {
  using T = F32Tile<D>;
  constexpr int BR = 32, KT = 64;
  __shared__ __attribute__((aligned(16))) float smem[4 * T::WORDS];       // two buffers of Q, dY
  __shared__ __attribute__((aligned(16))) float s_lse[2][BR], s_del[2][BR];
  __shared__ __attribute__((aligned(16))) int s_pos[2][BR];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, off = a.Tk - a.Tq;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const SpanSlot sl(a, w);
  const int k0 = sl.tile * KT;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  const KeySpan<KT> ks(a, k0, len);
  if (sl.part >= ks.parts) return;
  const int t0 = sl.part * ks.per * (64 / BR), t1 = min((sl.part + 1) * ks.per * (64 / BR), (ks.rows + BR - 1) / BR);
  const int kw = k0 + wave * 16, j = kw + n;
  f32x4 kf[T::NS], vf[T::NS];
  {
    const long long jj = max(0, min(j, len - 1));
    const float* kp = (const float*)a.k + b * a.ks[0] + hk * a.ks[2] + jj * a.ks[1];
    const float* vp = (const float*)a.v + b * a.vs[0] + hk * a.vs[2] + jj * a.vs[1];
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      kf[c] = *(const f32x4*)(kp + 16 * c + 4 * g);
      vf[c] = *(const f32x4*)(vp + 16 * c + 4 * g);
    }
  }
  const float sc = a.scale * kLog2e;
  f32x4 ok[T::NS], ov[T::NS];
#pragma unroll
  for (int t = 0; t < T::NS; ++t) ok[t] = ov[t] = zero4();
  const float* qb = (const float*)a.q + b * a.qs[0] + (long long)hk * G * a.qs[2];
  const float* gb = (const float*)a.dy + ((long long)b * a.Tq * a.Hq + hk * G) * D;
  F32Stage<D> st(tid);
  float x_lse = 0.f, x_del = 0.f;
  int x_pos = -1;
  RowMap rm(t0 * BR, G, a.g_magic);
  const auto load = [&](int t) {
    const int last = ks.rows - 1 - t * BR;
    st.load([&](int r, const float** pq, const float** pg) {
      int qi, qg;
      rm.at(min(r, last), &qi, &qg);
      qi += ks.i0;
      *pq = qb + qi * a.qs[1] + qg * a.qs[2];
      *pg = gb + ((long long)qi * a.Hq + qg) * D;
    });
    if (tid < BR) {
      int qi, qg;
      rm.at(min(tid, last), &qi, &qg);
      qi += ks.i0;
      const long long sr = ((long long)b * a.Hq + hk * G + qg) * a.Tq + qi;
      x_lse = a.lse[sr];
      x_del = a.delta[sr];
      x_pos = tid <= last ? qi + off : -1;
    }
  };
  const auto store = [&](int s) {
    st.store(smem + s * 2 * T::WORDS, smem + (s * 2 + 1) * T::WORDS);
    if (tid < BR) {
      s_lse[s][tid] = x_lse * kLog2e;
      s_del[s][tid] = x_del;
      s_pos[s][tid] = x_pos;
    }
  };
  if (t0 < t1) {
    load(t0);
    store(0);
  }
  lds_barrier();
  for (int t = t0; t < t1; ++t) {
    const int si = (t - t0) & 1;
    const float *sq = smem + si * 2 * T::WORDS, *sg = sq + T::WORDS;
    const int tp0 = rm.i0 + ks.i0 + off, tp1 = rm.last(BR - 1) + ks.i0 + off;
    if (t + 1 < t1) rm.advance(BR);
    load(min(t + 1, t1 - 1));
    if (tp1 >= kw && (tp0 - a.window < kw + 15 || kw < a.sinks)) {
      const bool all = (t + 1) * BR <= ks.rows && tp0 >= kw + 15 && (tp1 - kw < a.window || kw + 16 <= a.sinks);
      f32x4 pr[2], ds[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4 s = zero4(), dp = zero4();
#pragma unroll
        for (int c = 0; c < T::NS; ++c) {
          mma(s, ld_frag(sq + (16 * u + n) * T::LD + 16 * c, g), kf[c]);
          mma(dp, ld_frag(sg + (16 * u + n) * T::LD + 16 * c, g), vf[c]);
        }
        const f32x4 ls = *(const f32x4*)&s_lse[si][16 * u + 4 * g], dl = *(const f32x4*)&s_del[si][16 * u + 4 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool vis = all || attn_visible(s_pos[si][16 * u + 4 * g + e], j, a.window, a.sinks);
          pr[u][e] = vis ? exp2f(s[e] * sc - ls[e]) : 0.f;
          ds[u][e] = vis ? pr[u][e] * (dp[e] - dl[e]) : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < T::NS; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          mma(ov[c], ld_cols<T::LD>(sg, 16 * u, 16 * c + n, g), pr[u]);
          mma(ok[c], ld_cols<T::LD>(sq, 16 * u, 16 * c + n, g), ds[u]);
        }
    }
    store(si ^ 1);
    lds_barrier();
  }
  if (!key_seen(j, off, len, a.window, a.sinks)) {   // (0 times a query or dY that is not finite is NaN)
#pragma unroll
    for (int t = 0; t < T::NS; ++t) ok[t] = ov[t] = zero4();
  }
  if (ks.parts > 1) {                        // a span's sums, joined by win_dkv_join_kernel
    const long long slot = ((long long)b * a.Hkv + hk) * span_slots<KT>(a) + w;
    float* pk = a.part + (slot * 2 * KT + wave * 16 + n) * D + 4 * g;
#pragma unroll
    for (int t = 0; t < T::NS; ++t) {
      *(f32x4*)(pk + 16 * t) = ok[t];
      *(f32x4*)(pk + KT * D + 16 * t) = ov[t];
    }
    return;
  }
  if (j >= a.Tk) return;
  const long long row = ((long long)b * a.Tk + j) * a.Hkv + hk;
#pragma unroll
  for (int t = 0; t < T::NS; ++t) {
    *(f32x4*)((float*)a.dk + row * D + 16 * t + 4 * g) = ok[t] * a.scale;
    *(f32x4*)((float*)a.dv + row * D + 16 * t + 4 * g) = ov[t];
  }
}

// ---- shares of the work ----
// Rows a workgroup takes in the forward, keys a tile holds there and in the dk / dv kernel.
static int fwd_rows(int dtype) { return dtype == GDNX_DTYPE_BF16 ? 128 : 64; }
static int fwd_keys(int dtype) { return dtype == GDNX_DTYPE_BF16 ? 64 : 32; }
int win_dkv_keys(int dtype) { return dtype == GDNX_DTYPE_BF16 ? 128 : 64; }

// Parts that the rows' keys are cut into: as many as keep the workgroups within
// two a CU (so one from 257 workgroups on), each of at least four tiles (eight in
// bf16, whose tiles take less time beside the join, unless the workgroups are very
// few).  Forward in us, uncut / cut (bf16, d = 128 unless said): 2 x 200
// queries on 16584 keys, 16/2 heads 297 / 77; 2048 on 16384, 16/4 344 / 297;
// 4096 on 4096, 8/2 82 / 65; 16 on 4096, 8/8 109 / 16 (eight tiles: 21);
// float32, 200 on 8000, 8/4 762 / 89; 512 on 512, 16/4 54 / 32 (eight: 36).
// 2048 on 2048, window 512, 8/2 stays uncut: 18, cut by four tiles 22.
int win_attn_fwd_parts(int B, int Tq, int Tk, int Hq, int Hkv, int window, int sinks, int dtype) {
  const int G = Hq / Hkv, R = fwd_rows(dtype);
  const long long base = (((long long)Tq * G + R - 1) / R) * B * Hkv;
  const long long span = window > 0 ? (long long)window + sinks + (R - 1) / G + 1 : Tk, keys = span < Tk ? span : Tk;
  const long long tiles = (keys + fwd_keys(dtype) - 1) / fwd_keys(dtype);
  const int least = dtype == GDNX_DTYPE_BF16 && base > 32 ? 8 : 4;
  long long parts = 512 / base;
  if (parts > tiles / least) parts = tiles / least;
  return parts < 1 ? 1 : (int)parts;
}

// Tiles of keys see (tile + window) positions' rows, those with sinks every
// later one.  Ordinary tiles are cut only where the workgroups are too few to
// give every CU its three; the sinks' tiles, as long as the whole row, into
// spans of an ordinary tile's length.  Backward in us, uncut / cut (bf16,
// d = 128 unless said): 4 x 4096, window 1024, 16 sinks, 16/4 heads
// 1061 / 601; 8192 without a window, 16/4 1693 / 1044; 2048 without, 8/2
// 375 / 92; 5 x 1999, window 257, 3 sinks, 6/2, d = 64 257 / 67; float32,
// 2 x 4096, window 512, 4 sinks, 8/4 1785 / 695.
WinBwdPlan win_attn_bwd_plan(int B, int Tq, int Tk, int Hq, int Hkv, int window, int sinks, int dtype) {
  const int KT = win_dkv_keys(dtype);
  const long long G = Hq / Hkv, tiles = (Tk + KT - 1) / KT, heads = (long long)B * Hkv;
  const bool win = window > 0 && (long long)window + KT < Tk;
  const long long full = ((long long)Tq * G + 63) / 64;
  long long one = win ? (((long long)window + KT - 1) * G + 63) / 64 : full;
  if (one > full) one = full;
  const long long ns = sinks > 0 && win ? ((long long)sinks + KT - 1) / KT : 0;
  WinBwdPlan p;
  p.sink_tiles = (int)(ns < tiles ? ns : tiles);
  // all heads' steps: a triangle without a window, with one those of the tiles or, of fewer queries, of their rows
  long long seen = (tiles - p.sink_tiles) * one;
  const long long rows = full * (((long long)window + KT - 1) / KT + 1);
  if (seen > rows) seen = rows;
  const long long total = heads * (win ? seen + p.sink_tiles * full : tiles * full / 2);
  long long span = (total + 767) / 768;
  if (span < 8) span = 8;
  if (win && one <= 2 * span) span = span > one ? span : one;
  p.span = (int)span;
  p.tile_parts = (int)((one + span - 1) / span);
  p.sink_parts = (int)((full + span - 1) / span);
  return p;
}

template <int D> static int launch_fwd(const WinAttnArgs& a, hipStream_t stream) {
  const long long nt = ((long long)a.Tq * (a.Hq / a.Hkv) + 63) / 64;
  hipLaunchKernelGGL((win_fwd_f32_kernel<D>), dim3((unsigned)(nt * a.B * a.Hkv * a.parts)), dim3(256), 0, stream, a);
  const int rc = check_launch("win_fwd_f32_kernel");
  return rc ? rc : launch_win_join<float, D>(a, stream);
}

template <int D> static int launch_bwd(const WinAttnBwdArgs& a, hipStream_t stream) {
  const long long nt = ((long long)a.Tq * (a.Hq / a.Hkv) + 63) / 64, heads = (long long)a.B * a.Hkv;
  hipLaunchKernelGGL((win_dq_f32_kernel<D>), dim3((unsigned)(nt * heads * a.dq_parts)), dim3(256), 0, stream, a);
  int rc = check_launch("win_dq_f32_kernel");
  if (rc || (rc = launch_dq_join<float>(a, stream))) return rc;
  hipLaunchKernelGGL((win_dkv_f32_kernel<D>), dim3((unsigned)(span_slots<64>(a) * heads)), dim3(256), 0, stream, a);
  rc = check_launch("win_dkv_f32_kernel");
  return rc ? rc : launch_dkv_join<float, D, 64>(a, stream);
}

int win_attn_fwd_dispatch(const WinAttnArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16) return win_fwd_bf16_dispatch(a, stream);
  return a.D == 128 ? launch_fwd<128>(a, stream) : launch_fwd<64>(a, stream);
}

int win_attn_bwd_dispatch(const WinAttnBwdArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16) return win_bwd_bf16_dispatch(a, stream);
  return a.D == 128 ? launch_bwd<128>(a, stream) : launch_bwd<64>(a, stream);
}

}  // namespace gdnx
