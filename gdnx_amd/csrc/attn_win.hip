// Attention with a sliding window and sinks, forward and backward (gfx950):
// the kernels that serve every type and size.
//
//   P_ij = exp(s q_i.k_j - lse_i) over the visible j,  y_i = sum_j P_ij v_j
//   dV = P^T dY;  dP = dY V^T;  dS = P o (dP - delta),  delta_i = dY_i.Y_i;
//   dQ = s dS K;  dK = s dS^T Q, both summed over a key head's query heads.
//
// One wave owns 16 queries (forward, dq) or 16 keys (dk, dv).  The scores are
// formed transposed to what they are contracted over next, so that a score
// tile's accumulators are the next product's operand: S^T = K Q^T feeds
// O^T = V^T P^T and dQ^T = K^T dS^T; S = Q K^T feeds dV^T = dY^T P and
// dK^T = Q^T dS.  Softmax statistics, sums and products are float32.
#include "attn_common.hpp"

namespace gdnx {

// Fragment over rows kb.. of a row-major LDS tile, column c of the lane.
template <int LD> __device__ __forceinline__ bf16x8 ld_frag_rows(const bf16* t, int kb, int c, int g) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = t[(kb + 4 * g + i) * LD + c];
    r[4 + i] = t[(kb + 16 + 4 * g + i) * LD + c];
  }
  return r;
}
template <int LD> __device__ __forceinline__ f32x4 ld_frag_rows(const float* t, int kb, int c, int g) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = t[(kb + 4 * g + i) * LD + c];
  return r;
}

// Rows [r0, r0 + N) of a strided [rows][D] matrix into an LDS tile; rows
// outside [0, end) are zero, so that what padding holds never enters a product.
template <typename CT, int D, int N, int LD, int TH>
__device__ __forceinline__ void stage_rows(CT* dst, const CT* src, long long stride, int r0, int end, int tid) {
  constexpr int EPU = 16 / sizeof(CT), UPR = D / EPU;
#pragma unroll
  for (int u = tid; u < N * UPR; u += TH) {
    const int r = u / UPR, c = (u % UPR) * EPU;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r0 + r >= 0 && r0 + r < end) x = *(const uint4*)(src + (long long)(r0 + r) * stride + c);
    *(uint4*)(dst + r * LD + c) = x;
  }
}

// A wave's 16 rows as fragments (row n of the lane); rows outside are zero.
template <typename CT, int D>
__device__ __forceinline__ void load_row_frags(typename FragT<CT>::type* f, const CT* src, long long stride, int row,
                                               bool ok, int g) {
  constexpr int KS = FragT<CT>::KSTEP;
#pragma unroll
  for (int s = 0; s < D / KS; ++s) {
    if (ok) f[s] = ld_frag(src + (long long)row * stride + s * KS, g);
    else f[s] = typename FragT<CT>::type{};
  }
}

template <typename CT, int D> struct WinTile {
  static constexpr int BK = 32, NW = 4, BQ = 16 * NW, TH = 64 * NW, LD = D + 16 / (int)sizeof(CT);
  static constexpr int KS = FragT<CT>::KSTEP, NS = D / KS, TPS = FragT<CT>::TPS, NT = D / 16;
};

template <typename CT, int D>
__global__ void __launch_bounds__(256) win_attn_fwd_kernel(WinAttnArgs a) {
  using W = WinTile<CT, D>;
  typedef typename FragT<CT>::type Frag;
  __shared__ __attribute__((aligned(16))) CT sk[W::BK * W::LD], sv[W::BK * W::LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int nqt = (a.Tq + W::BQ - 1) / W::BQ, G = a.Hq / a.Hkv;
  // work order: a key head's query heads and tiles are neighbours (one XCD's L2)
  const int w = xcd_remap(blockIdx.x, gridDim.x);
  const int h = (w / nqt) % a.Hq, b = w / nqt / a.Hq, i0 = (w % nqt) * W::BQ, hk = h / G;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const CT* qb = (const CT*)a.q + b * a.qs[0] + h * a.qs[2];
  const CT* kb = (const CT*)a.k + b * a.ks[0] + hk * a.ks[2];
  const CT* vb = (const CT*)a.v + b * a.vs[0] + hk * a.vs[2];
  const int i = i0 + wave * 16 + n;
  const int p = i < a.Tq && i + off < len ? i + off : -1;
  Frag qf[W::NS];
  load_row_frags<CT, D>(qf, qb, a.qs[1], i, p >= 0, g);
  const float sc = a.scale * kLog2e;
  f32x4 o[W::NT];
#pragma unroll
  for (int t = 0; t < W::NT; ++t) o[t] = zero4();
  float m = -INFINITY, l = 0.f;
  const KeyTiles<W::BK> kt(i0 + off, min(i0 + W::BQ, a.Tq) - 1 + off, len, a.window, a.sinks);
  for (int it = 0; it < kt.count; ++it) {
    const int j0 = kt.start(it);
    __syncthreads();
    stage_rows<CT, D, W::BK, W::LD, W::TH>(sk, kb, a.ks[1], j0, len, tid);
    stage_rows<CT, D, W::BK, W::LD, W::TH>(sv, vb, a.vs[1], j0, len, tid);
    __syncthreads();
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = zero4();
#pragma unroll
      for (int c = 0; c < W::NS; ++c) mma(s[u], ld_frag(sk + (16 * u + n) * W::LD + c * W::KS, g), qf[c]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[u][e] = attn_visible(p, j0 + 16 * u + 4 * g + e, a.window, a.sinks) ? s[u][e] * sc : -INFINITY;
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
    for (int t = 0; t < W::NT; ++t) {
      o[t] *= f;
#pragma unroll
      for (int c = 0; c < W::BK / W::KS; ++c)
        mma(o[t], ld_frag_rows<W::LD>(sv, c * W::KS, 16 * t + n, g),
            acc_frag((CT*)nullptr, s[c * W::TPS], s[c * W::TPS + W::TPS - 1]));
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (i >= a.Tq) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // (a NaN sum stays one)
  CT* yb = (CT*)a.y + (((long long)b * a.Tq + i) * a.Hq + h) * D;
#pragma unroll
  for (int t = 0; t < W::NT; ++t)
    st4(yb + 16 * t + 4 * g, o[t][0] * inv, o[t][1] * inv, o[t][2] * inv, o[t][3] * inv);
  if (g == 0 && a.lse) a.lse[((long long)b * a.Hq + h) * a.Tq + i] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// dq, and delta for the dk / dv kernel
template <typename CT, int D>
__global__ void __launch_bounds__(256) win_attn_dq_kernel(WinAttnBwdArgs a) {
  using W = WinTile<CT, D>;
  typedef typename FragT<CT>::type Frag;
  __shared__ __attribute__((aligned(16))) CT sk[W::BK * W::LD], sv[W::BK * W::LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int nqt = (a.Tq + W::BQ - 1) / W::BQ, G = a.Hq / a.Hkv;
  const int w = xcd_remap(blockIdx.x, gridDim.x);
  const int h = (w / nqt) % a.Hq, b = w / nqt / a.Hq, i0 = (w % nqt) * W::BQ, hk = h / G;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const CT* kb = (const CT*)a.k + b * a.ks[0] + hk * a.ks[2];
  const CT* vb = (const CT*)a.v + b * a.vs[0] + hk * a.vs[2];
  const int i = i0 + wave * 16 + n;
  const int p = i < a.Tq && i + off < len ? i + off : -1;
  const long long row = ((long long)b * a.Tq + i) * a.Hq + h, srow = ((long long)b * a.Hq + h) * a.Tq + i;
  Frag qf[W::NS], gf[W::NS];
  load_row_frags<CT, D>(qf, (const CT*)a.q + b * a.qs[0] + h * a.qs[2], a.qs[1], i, p >= 0, g);
  load_row_frags<CT, D>(gf, (const CT*)a.dy + row * D, 0, 0, p >= 0, g);
  float delta = 0.f, lse = 0.f;
  {
    Frag yf[W::NS];
    load_row_frags<CT, D>(yf, (const CT*)a.y + row * D, 0, 0, p >= 0, g);
#pragma unroll
    for (int s = 0; s < W::NS; ++s)
#pragma unroll
      for (int e = 0; e < (int)(sizeof(Frag) / sizeof(CT)); ++e) delta += to_f(gf[s][e]) * to_f(yf[s][e]);
    delta += __shfl_xor(delta, 16, 64);
    delta += __shfl_xor(delta, 32, 64);
    if (g == 0 && i < a.Tq) a.delta[srow] = delta;
    if (p >= 0) lse = a.lse[srow] * kLog2e;
  }
  const float sc = a.scale * kLog2e;
  f32x4 o[W::NT];
#pragma unroll
  for (int t = 0; t < W::NT; ++t) o[t] = zero4();
  const KeyTiles<W::BK> kt(i0 + off, min(i0 + W::BQ, a.Tq) - 1 + off, len, a.window, a.sinks);
  for (int it = 0; it < kt.count; ++it) {
    const int j0 = kt.start(it);
    __syncthreads();
    stage_rows<CT, D, W::BK, W::LD, W::TH>(sk, kb, a.ks[1], j0, len, tid);
    stage_rows<CT, D, W::BK, W::LD, W::TH>(sv, vb, a.vs[1], j0, len, tid);
    __syncthreads();
    f32x4 ds[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 s = zero4(), dp = zero4();
#pragma unroll
      for (int c = 0; c < W::NS; ++c) {
        mma(s, ld_frag(sk + (16 * u + n) * W::LD + c * W::KS, g), qf[c]);
        mma(dp, ld_frag(sv + (16 * u + n) * W::LD + c * W::KS, g), gf[c]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        ds[u][e] = attn_visible(p, j0 + 16 * u + 4 * g + e, a.window, a.sinks)
                       ? exp2f(s[e] * sc - lse) * (dp[e] - delta) * a.scale : 0.f;
    }
#pragma unroll
    for (int t = 0; t < W::NT; ++t)
#pragma unroll
      for (int c = 0; c < W::BK / W::KS; ++c)
        mma(o[t], ld_frag_rows<W::LD>(sk, c * W::KS, 16 * t + n, g),
            acc_frag((CT*)nullptr, ds[c * W::TPS], ds[c * W::TPS + W::TPS - 1]));
  }
  if (i >= a.Tq) return;
  CT* qo = (CT*)a.dq + row * D;
#pragma unroll
  for (int t = 0; t < W::NT; ++t) st4(qo + 16 * t + 4 * g, o[t][0], o[t][1], o[t][2], o[t][3]);
}

// dk, dv of 64 keys: the group's query heads in turn, each over the queries
// that see some of the keys
template <typename CT, int D>
__global__ void __launch_bounds__(256) win_attn_dkv_kernel(WinAttnBwdArgs a) {
  using W = WinTile<CT, D>;
  typedef typename FragT<CT>::type Frag;
  constexpr int BQ = W::BK, BKV = W::BQ;      // 32 queries a step, 64 keys a workgroup
  __shared__ __attribute__((aligned(16))) CT sq[BQ * W::LD], sg[BQ * W::LD];
  __shared__ __attribute__((aligned(16))) float slse[BQ], sdel[BQ];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int nkt = (a.Tk + BKV - 1) / BKV, G = a.Hq / a.Hkv;
  const int w = xcd_remap(blockIdx.x, gridDim.x);
  const int hk = (w / nkt) % a.Hkv, b = w / nkt / a.Hkv, k0 = (w % nkt) * BKV;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const int j = k0 + wave * 16 + n;
  Frag kf[W::NS], vf[W::NS];
  load_row_frags<CT, D>(kf, (const CT*)a.k + b * a.ks[0] + hk * a.ks[2], a.ks[1], j, j < len, g);
  load_row_frags<CT, D>(vf, (const CT*)a.v + b * a.vs[0] + hk * a.vs[2], a.vs[1], j, j < len, g);
  const float sc = a.scale * kLog2e;
  f32x4 ok[W::NT], ov[W::NT];
#pragma unroll
  for (int t = 0; t < W::NT; ++t) ok[t] = ov[t] = zero4();
  const int pe = k0 < len ? last_query<BKV>(k0, len, a.window, a.sinks) : 0;
  for (int hg = 0; hg < G; ++hg) {
    const int h = hk * G + hg;
    const CT* qb = (const CT*)a.q + b * a.qs[0] + h * a.qs[2];
    const CT* gb = (const CT*)a.dy + ((long long)b * a.Tq * a.Hq + h) * D;
    const float* lb = a.lse + ((long long)b * a.Hq + h) * a.Tq;
    const float* db = a.delta + ((long long)b * a.Hq + h) * a.Tq;
    for (int p0 = max(k0, off); p0 < pe; p0 += BQ) {
      const int i0 = p0 - off;
      __syncthreads();
      stage_rows<CT, D, BQ, W::LD, W::TH>(sq, qb, a.qs[1], i0, len - off, tid);
      stage_rows<CT, D, BQ, W::LD, W::TH>(sg, gb, (long long)a.Hq * D, i0, len - off, tid);
      if (tid < BQ) {
        const bool in = i0 + tid < a.Tq && p0 + tid < len;
        slse[tid] = in ? lb[i0 + tid] * kLog2e : 0.f;
        sdel[tid] = in ? db[i0 + tid] : 0.f;
      }
      __syncthreads();
      f32x4 pr[2], ds[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4 s = zero4(), dp = zero4();
#pragma unroll
        for (int c = 0; c < W::NS; ++c) {
          mma(s, ld_frag(sq + (16 * u + n) * W::LD + c * W::KS, g), kf[c]);
          mma(dp, ld_frag(sg + (16 * u + n) * W::LD + c * W::KS, g), vf[c]);
        }
        const f32x4 ls = *(const f32x4*)&slse[16 * u + 4 * g], dl = *(const f32x4*)&sdel[16 * u + 4 * g];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p = p0 + 16 * u + 4 * g + e;
          const bool vis = attn_visible(p < len ? p : -1, j, a.window, a.sinks);
          pr[u][e] = vis ? exp2f(s[e] * sc - ls[e]) : 0.f;
          ds[u][e] = vis ? pr[u][e] * (dp[e] - dl[e]) * a.scale : 0.f;
        }
      }
#pragma unroll
      for (int t = 0; t < W::NT; ++t)
#pragma unroll
        for (int c = 0; c < BQ / W::KS; ++c) {
          mma(ov[t], ld_frag_rows<W::LD>(sg, c * W::KS, 16 * t + n, g),
              acc_frag((CT*)nullptr, pr[c * W::TPS], pr[c * W::TPS + W::TPS - 1]));
          mma(ok[t], ld_frag_rows<W::LD>(sq, c * W::KS, 16 * t + n, g),
              acc_frag((CT*)nullptr, ds[c * W::TPS], ds[c * W::TPS + W::TPS - 1]));
        }
    }
  }
  if (j >= a.Tk) return;
  const long long row = ((long long)b * a.Tk + j) * a.Hkv + hk;
#pragma unroll
  for (int t = 0; t < W::NT; ++t) {
    st4((CT*)a.dk + row * D + 16 * t + 4 * g, ok[t][0], ok[t][1], ok[t][2], ok[t][3]);
    st4((CT*)a.dv + row * D + 16 * t + 4 * g, ov[t][0], ov[t][1], ov[t][2], ov[t][3]);
  }
}

template <typename CT, int D> static int launch_fwd(const WinAttnArgs& a, hipStream_t stream) {
  const long long nqt = (a.Tq + 63) / 64;
  hipLaunchKernelGGL((win_attn_fwd_kernel<CT, D>), dim3((unsigned)(nqt * a.B * a.Hq)), dim3(256), 0, stream, a);
  return check_launch("win_attn_fwd_kernel");
}

template <typename CT, int D> static int launch_bwd(const WinAttnBwdArgs& a, hipStream_t stream) {
  const long long nqt = (a.Tq + 63) / 64, nkt = (a.Tk + 63) / 64;
  hipLaunchKernelGGL((win_attn_dq_kernel<CT, D>), dim3((unsigned)(nqt * a.B * a.Hq)), dim3(256), 0, stream, a);
  const int rc = check_launch("win_attn_dq_kernel");
  if (rc) return rc;
  hipLaunchKernelGGL((win_attn_dkv_kernel<CT, D>), dim3((unsigned)(nkt * a.B * a.Hkv)), dim3(256), 0, stream, a);
  return check_launch("win_attn_dkv_kernel");
}

int win_attn_fwd_dispatch(const WinAttnArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16) return win_fwd_bf16_dispatch(a, stream);
  return a.D == 128 ? launch_fwd<float, 128>(a, stream) : launch_fwd<float, 64>(a, stream);
}

int win_attn_bwd_dispatch(const WinAttnBwdArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16) return win_bwd_bf16_dispatch(a, stream);
  return a.D == 128 ? launch_bwd<float, 128>(a, stream) : launch_bwd<float, 64>(a, stream);
}

}  // namespace gdnx
