// Short causal convolution along a sequence, a filter of W taps for every
// channel, with its activation (gfx950).
//
//   u_t = bias + sum_k w[W-1-k] x_{t-k},   y_t = u_t sigmoid(u_t)  (or u_t)
//   du_t = dy_t s (1 + u_t (1 - s)),  s = sigmoid(u_t);
//   dx_t = sum_k w[W-1-k] du_{t+k},  dw[W-1-k] = sum_t du_t x_{t-k},  dbias = sum_t du_t
//
// x before a sequence's first token is its state, the last W - 1 inputs.
// Channels are contiguous: a lane takes a few of them
// and walks along the tokens with the last W - 1 inputs in registers, so x is
// read once but for the W - 1 rows before each span.  Sums are float32.
#include <type_traits>

#include "gdnx_internal.hpp"
#include "packed_rows.hpp"

namespace gdnx {

namespace {

// V channels of a row as they lie in memory; rows may have any alignment.
template <typename CT, int V> struct Raw {
  static constexpr int WORDS = V * (int)sizeof(CT) / 4;
  typedef CT T __attribute__((ext_vector_type(V)));
  T x;
  __device__ __forceinline__ void load(const CT* p) { __builtin_memcpy(&x, p, sizeof(x)); }
  __device__ __forceinline__ void get(float* out) const {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = to_f(x[e]);
  }
  __device__ __forceinline__ void get(float* out, bool there) const {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = there ? to_f(x[e]) : 0.f;
  }
};
template <typename CT> struct Raw<CT, 1> {
  CT x;
  __device__ __forceinline__ void load(const CT* p) { x = *p; }
  __device__ __forceinline__ void get(float* out) const { out[0] = to_f(x); }
  __device__ __forceinline__ void get(float* out, bool there) const { out[0] = there ? to_f(x) : 0.f; }
};
template <typename CT, int V> __device__ __forceinline__ void st_chan(CT* p, const float* in) {
  CT x[V];
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = from_f<CT>(in[e]);
  __builtin_memcpy(p, x, sizeof(x));
}
// (past the caches: nothing here reads it again)
template <typename CT, int V> __device__ __forceinline__ void st_chan_nt(CT* p, const float* in) {
  typedef CT T __attribute__((ext_vector_type(V), aligned(sizeof(CT))));
  if constexpr (V == 1) {
    __builtin_nontemporal_store(from_f<CT>(in[0]), p);
  } else {
    T x;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = from_f<CT>(in[e]);
    __builtin_nontemporal_store(x, (T*)p);
  }
}
template <int V> __device__ __forceinline__ void zero_chan(float* x) {
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = 0.f;
}
template <int W, int V> __device__ __forceinline__ void shift(float (*x)[V]) {
#pragma unroll
  for (int k = W - 1; k > 0; --k)
#pragma unroll
    for (int e = 0; e < V; ++e) x[k][e] = x[k - 1][e];
}

// w[k] multiplies x_{t-k}
template <typename WT, int W, int V>
__device__ __forceinline__ void ld_weights(float (*w)[V], float* bias, const ConvArgs& a, int c) {
  WT x[V * W], b[V];
  __builtin_memcpy(x, (const WT*)a.weight + (long long)c * W, sizeof(x));
  if (a.bias) __builtin_memcpy(b, (const WT*)a.bias + c, sizeof(b));
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = to_f(x[e * W + W - 1 - k]);
    bias[e] = a.bias ? to_f(b[e]) : 0.f;
  }
}
template <int W, int V> __device__ __forceinline__ void ld_weights(float (*w)[V], float* bias, const ConvArgs& a, int c) {
  if (a.wdtype == GDNX_DTYPE_BF16) ld_weights<bf16, W, V>(w, bias, a, c);
  else ld_weights<float, W, V>(w, bias, a, c);
}

// 1 / (1 + e^-u): the reciprocal is the hardware's, of one unit in the last
// place (a division takes ten instructions of them, a third of the forward's)
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __expf(-u)); }

template <int W, int V>
__device__ __forceinline__ void conv_out(float* y, const float (*w)[V], const float* bias, const float (*x)[V], int silu) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float u = bias[e];
#pragma unroll
    for (int k = 0; k < W; ++k) u = fmaf(w[k][e], x[k][e], u);
    y[e] = silu ? u * sigmoid(u) : u;
  }
}

// A thread's channels and tokens: lanes of a workgroup side by side on the
// channels, its 256 >> lx_log rows of them on spans of tokens.  Where V does
// not divide C, the last channels are taken twice, by two lanes that store
// the same.
template <int V> struct ConvPlace {
  int c, b, t0;
  bool there;
  __device__ __forceinline__ static int channel(const ConvArgs& a, int unit) { return min(unit * V, a.C - V); }
  __device__ __forceinline__ ConvPlace(const ConvArgs& a) {
    const int lx = threadIdx.x & ((1 << a.lx_log) - 1), ly = threadIdx.x >> a.lx_log;
    int w = blockIdx.x;
    const int g = w % a.groups; w /= a.groups;
    b = w / a.blocks;
    const int unit = (g << a.lx_log) + lx;
    c = channel(a, unit);
    t0 = ((w - b * a.blocks) * (256 >> a.lx_log) + ly) * a.span;
    there = unit * V < a.C && t0 < a.T;
  }
};

// Rows of a sequence of `len` tokens.  Loads are made whatever t is, from the
// nearest valid token, so that many are in flight; what they give is masked.
template <typename CT, int V> struct ConvRow {
  const CT *x, *state;
  long long xt;
  int len, last, W1, C;
  __device__ __forceinline__ ConvRow(const ConvArgs& a, int b, int c)
      : x((const CT*)a.x + b * a.xs[0] + c), state(a.state ? (const CT*)a.state + (long long)b * (a.W - 1) * a.C + c : nullptr),
        xt(a.xs[1]), W1(a.W - 1), C(a.C) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    last = max(len - 1, 0);
  }
  __device__ __forceinline__ Raw<CT, V> load(int t) const {
    Raw<CT, V> r;
    r.load(x + min(t, last) * xt);
    return r;
  }
  // any t < len: the state before token 0, zeros where there is none
  __device__ __forceinline__ void at(float* out, int t) const {
    Raw<CT, V> r;
    if (t >= 0) {
      r.load(x + min(t, last) * xt);
      r.get(out, len > 0);
    } else if (state) {
      r.load(state + (long long)(W1 + t) * C);
      r.get(out);
    } else {
      zero_chan<V>(out);
    }
  }
};

}  // namespace

template <typename CT, int W, int V> __global__ void __launch_bounds__(256) conv_fwd_kernel(ConvArgs a) {
  constexpr int U = 4;
  const ConvPlace<V> pl(a);
  if (!pl.there) return;
  const ConvRow<CT, V> row(a, pl.b, pl.c);
  float w[W][V], bias[V], x[W][V];
  Raw<CT, V> next[U];
#pragma unroll
  for (int i = 0; i < U; ++i) next[i] = row.load(pl.t0 + i);
  ld_weights<W, V>(w, bias, a, pl.c);
#pragma unroll
  for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
  const int t1 = min(pl.t0 + a.span, a.T);
  CT* y = (CT*)a.y + ((long long)pl.b * a.T + pl.t0) * a.C + pl.c;
  for (int t = pl.t0; t < t1; t += U) {
    Raw<CT, V> in[U];
#pragma unroll
    for (int i = 0; i < U; ++i) in[i] = next[i];
#pragma unroll
    for (int i = 0; i < U; ++i) next[i] = row.load(t + U + i);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      shift<W, V>(x);
      in[i].get(x[0]);
      float o[V];
      conv_out<W, V>(o, w, bias, x, a.silu);
      if (t + i >= row.len) zero_chan<V>(o);
      if (t + i < t1) st_chan<CT, V>(y, o);
      y += a.C;
    }
  }
  if (a.state_out && pl.t0 == 0) {           // the last W - 1 inputs before len
    CT* so = (CT*)a.state_out + (long long)pl.b * (W - 1) * a.C + pl.c;
#pragma unroll
    for (int m = 0; m < W - 1; ++m) {
      float s[V];
      row.at(s, row.len - (W - 1) + m);
      st_chan<CT, V>(so + (long long)m * a.C, s);
    }
  }
}

// The gradients of a span in one walk along its tokens and the W - 1 behind
// it: du_t goes into the W sums dx_{t-k} that wait for it, the oldest of which
// is then whole.  Filter gradients are summed over the span, then over the
// workgroup, and stored [block][W + 1][C] for the join.
template <typename CT, int W, int V> __global__ void __launch_bounds__(256) conv_bwd_kernel(ConvArgs a) {
  constexpr int U = 4;
  __shared__ float sh[256 * V];
  const ConvPlace<V> pl(a);
  float dw[W][V], db[V];
#pragma unroll
  for (int k = 0; k < W; ++k) zero_chan<V>(dw[k]);
  zero_chan<V>(db);
  if (pl.there) {
    const ConvRow<CT, V> row(a, pl.b, pl.c);
    const long long at = (long long)pl.b * a.T * a.C + pl.c, sat = (long long)pl.b * (W - 1) * a.C + pl.c;
    const CT* dy = (const CT*)a.dy + at;
    CT* dx = (CT*)a.dx + at;
    float w[W][V], bias[V], x[W][V], acc[W][V];
    Raw<CT, V> nx[U], ng[U];
    const auto ask = [&](int t) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        nx[i] = row.load(t + i);
        ng[i].load(dy + (long long)min(t + i, row.last) * a.C);
      }
    };
    ask(pl.t0);
    ld_weights<W, V>(w, bias, a, pl.c);
#pragma unroll
    for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
#pragma unroll
    for (int k = 0; k < W; ++k) zero_chan<V>(acc[k]);
    const int t1 = min(pl.t0 + a.span, a.T);
    // token t's du from its row and gradient, into the sums that wait for it
    const auto token = [&](const Raw<CT, V>& rx, const Raw<CT, V>& rg, int t, bool mine) {
      const bool there = t < row.len;
      float g[V];
      shift<W, V>(x);
      shift<W, V>(acc);
      rx.get(x[0], there);
      rg.get(g, there);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float du = g[e];
        if (a.silu) {
          float u = bias[e];
#pragma unroll
          for (int k = 0; k < W; ++k) u = fmaf(w[k][e], x[k][e], u);
          const float s = sigmoid(u);
          du *= s * fmaf(u, 1.f - s, 1.f);
          if (!there) du = 0.f;              // (u may be no number)
        }
        acc[0][e] = w[0][e] * du;
#pragma unroll
        for (int k = 1; k < W; ++k) acc[k][e] = fmaf(w[k][e], du, acc[k][e]);
        if (mine) {
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k][e] = fmaf(du, x[k][e], dw[k][e]);
          db[e] += du;
        }
      }
      const int tau = t - (W - 1);               // dx of this token is whole
      if (tau >= t1 || (tau < pl.t0 && pl.t0 > 0)) return;
      const int m = tau - row.len + W - 1;       // its place in the state that is handed on
      if (a.dstate_out && tau < row.len && m >= 0) {
        Raw<CT, V> so;
        float s[V];
        so.load((const CT*)a.dstate_out + sat + (long long)m * a.C);
        so.get(s);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[W - 1][e] += s[e];
      }
      if (tau >= 0) st_chan_nt<CT, V>(dx + (long long)tau * a.C, acc[W - 1]);
      else if (a.dstate) st_chan<CT, V>((CT*)a.dstate + sat + (long long)(tau + W - 1) * a.C, acc[W - 1]);
    };
    int t = pl.t0;
    for (; t < t1; t += U) {
      Raw<CT, V> rx[U], rg[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        rx[i] = nx[i];
        rg[i] = ng[i];
      }
      ask(t + U);
#pragma unroll
      for (int i = 0; i < U; ++i) token(rx[i], rg[i], t + i, true);
    }
    // the tokens behind, whose filter gradients are another span's (behind the row's end there is nothing)
    for (; t < t1 + W - 1; t += U) {
      Raw<CT, V> rx[U], rg[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        rx[i] = nx[i];
        rg[i] = ng[i];
      }
      ask(t + U);
#pragma unroll
      for (int i = 0; i < U; ++i) token(rx[i], rg[i], t + i, false);
    }
  }
  // the workgroup's rows summed in order, a tap at a time
  const int lx = threadIdx.x & ((1 << a.lx_log) - 1), ly = threadIdx.x >> a.lx_log, rows = 256 >> a.lx_log;
  float* out = a.part + (long long)(blockIdx.x / a.groups) * (W + 1) * a.C;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) sh[((ly << a.lx_log) + lx) * V + e] = k < W ? dw[k < W ? k : 0][e] : db[e];
    __syncthreads();
    for (int u = threadIdx.x; u < V << a.lx_log; u += 256) {
      const int unit = ((blockIdx.x % a.groups) << a.lx_log) + u / V;
      float s = 0.f;
      for (int r = 0; r < rows; ++r) s += sh[(r << a.lx_log) * V + u];
      if (unit * V < a.C) out[(long long)k * a.C + ConvPlace<V>::channel(a, unit) + u % V] = s;
    }
    __syncthreads();
  }
}

// Blocks' filter gradients summed in order: [blocks][W + 1][C] -> dweight [C,W],
// dbias [C].  A workgroup takes 64 of the columns, a wave a quarter of the blocks.
__global__ void __launch_bounds__(256) conv_join_kernel(ConvArgs a, int blocks) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long u = (long long)blockIdx.x * 64 + lane, n = (long long)(a.W + 1) * a.C;
  const int per = (blocks + 3) / 4, i1 = min(blocks, (wave + 1) * per);
  float s = 0.f;
  if (u < n) {
#pragma unroll 8
    for (int i = wave * per; i < i1; ++i) s += a.part[i * n + u];
  }
  sh[wave][lane] = s;
  __syncthreads();
  if (wave || u >= n) return;
  s = sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane];
  const int k = (int)(u / a.C), c = (int)(u % a.C);
  void* to = k < a.W ? a.dweight : a.dbias;
  if (!to) return;
  const long long at = k < a.W ? (long long)c * a.W + a.W - 1 - k : c;
  if (a.wdtype == GDNX_DTYPE_BF16) ((bf16*)to)[at] = (bf16)s;
  else ((float*)to)[at] = s;
}

// Packed rows of unlike lengths, each with a slot of the state pool: a wave
// takes a span of one row's tokens (row_item).  The row's first wave alone
// reads the old state, before it writes the new one.  FULL: V divides C;
// otherwise the last lane takes what is left, a channel at a time.
template <typename CT, int W, int V, bool FULL> __global__ void __launch_bounds__(256) conv_packed_kernel(ConvPackedArgs p) {
  constexpr int U = 4;
  const ConvArgs& a = p.a;
  const int lane = threadIdx.x & 63;
  const int item = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / a.groups) * 4 + (threadIdx.x >> 6));
  int i, o0, n, tile;
  if (!row_item(p.offsets, p.n, p.N, 1, a.span, item, lane, &i, &o0, &n, &tile)) return;
  const int t0 = tile * a.span;
  if (t0 >= n && tile > 0) return;
  const int slot = p.slots ? p.slots[i] : i, to = p.to_slots ? p.to_slots[i] : slot;
  const bool live = slot >= 0 && slot < p.n_slots, store = live && to >= 0 && to < p.n_slots;
  const int c0 = ((int)(blockIdx.x % a.groups) * 64 + lane) * V;
  if (c0 >= a.C) return;
  const auto channels = [&](auto width, int c) {       // `width` channels from c on
    constexpr int N = decltype(width)::value;
    const CT* x = (const CT*)a.x + o0 * a.xs[1] + c;
    const CT* state = (const CT*)a.state + (long long)(live ? slot : 0) * (W - 1) * a.C + c;
    const int t1 = min(t0 + a.span, n);
    Raw<CT, N> next[U];
    const auto ask = [&](int t) {                      // (a row without tokens reads its state's first row)
#pragma unroll
      for (int e = 0; e < U; ++e) next[e].load(n > 0 ? x + min(t + e, n - 1) * a.xs[1] : state);
    };
    ask(t0);
    const auto at = [&](int t) {                       // t < n: an input, or the state's
      Raw<CT, N> r;
      r.load(t >= 0 ? x + t * a.xs[1] : state + (long long)(W - 1 + t) * a.C);
      return r;
    };
    float w[W][N], bias[N], xw[W][N];
    Raw<CT, N> before[W - 1], handed[W - 1];
#pragma unroll
    for (int k = 1; k < W; ++k) before[k - 1] = at(t0 - k);
    if (tile == 0) {
#pragma unroll
      for (int m = 0; m < W - 1; ++m) handed[m] = at(n - (W - 1) + m);
    }
    ld_weights<W, N>(w, bias, a, c);
    if (tile == 0 && store) {
      CT* so = (CT*)a.state_out + (long long)to * (W - 1) * a.C + c;
#pragma unroll
      for (int m = 0; m < W - 1; ++m) __builtin_memcpy(so + (long long)m * a.C, &handed[m].x, sizeof(handed[m].x));
    }
#pragma unroll
    for (int k = 1; k < W; ++k) before[k - 1].get(xw[k - 1]);
    CT* y = (CT*)a.y + ((long long)o0 + t0) * a.C + c;
    for (int t = t0; t < t1; t += U) {
      Raw<CT, N> in[U];
#pragma unroll
      for (int e = 0; e < U; ++e) in[e] = next[e];
      if (t + U < t1) ask(t + U);
#pragma unroll
      for (int e = 0; e < U; ++e) {
        shift<W, N>(xw);
        in[e].get(xw[0]);
        float o[N];
        conv_out<W, N>(o, w, bias, xw, a.silu);
        if (!live) zero_chan<N>(o);
        if (t + e < t1) st_chan<CT, N>(y, o);
        y += a.C;
      }
    }
  };
  if (FULL || c0 + V <= a.C) {
    channels(std::integral_constant<int, V>{}, c0);
  } else {
    for (int c = c0; c < a.C; ++c) channels(std::integral_constant<int, 1>{}, c);
  }
}

// Channels a lane; one where there are fewer.  Forward: 16 bytes, 8 from W = 5
// on.  Backward, which holds four rows of W for a channel: four (eight of bf16
// 165 us in the training step of 4 x 4096 tokens and 6144 channels, four 143),
// two in float32 from W = 5 on.
template <typename CT, int W> struct ConvLanes {
  static constexpr int FWD = 16 / sizeof(CT) / (W <= 4 ? 1 : 2), BWD = FWD < 4 ? FWD : 4;
};
static int conv_lanes(int C, int W, int dtype, bool bwd) {
  const int fwd = (dtype == GDNX_DTYPE_BF16 ? 8 : 4) / (W <= 4 ? 1 : 2), V = bwd && fwd > 4 ? 4 : fwd;
  return C < V ? 1 : V;
}

// Lanes on the channels (a power of two up to 64), groups of them, tokens a
// thread takes and blocks of a row.
static void conv_shape(ConvArgs& a, int V) {
  const int units = (a.C + V - 1) / V;
  a.lx_log = 0;
  while ((1 << a.lx_log) < units && a.lx_log < 6) ++a.lx_log;
  a.groups = (units + (1 << a.lx_log) - 1) >> a.lx_log;
  const int rows = 256 >> a.lx_log;
  for (a.span = 64;; a.span /= 2) {
    a.blocks = (a.T + rows * a.span - 1) / (rows * a.span);
    if (a.span == 8 || (long long)a.blocks * a.B * a.groups >= 1024) break;
  }
}

static ConvArgs shaped(int B, int T, int C, int W, int dtype, bool bwd) {
  ConvArgs a{};
  a.B = B; a.T = T; a.C = C; a.W = W;
  conv_shape(a, conv_lanes(C, W, dtype, bwd));
  return a;
}
long long conv_bwd_blocks(int B, int T, int C, int W, int dtype) {
  return (long long)shaped(B, T, C, W, dtype, true).blocks * B;
}
long long conv_groups(int B, int T, int C, int W, int dtype) {      // (the backward's lanes are the narrower ones)
  const ConvArgs a = shaped(B, T, C, W, dtype, true);
  return (long long)a.blocks * B * a.groups;
}

template <typename CT, int W, int V> static int launch_fwd(ConvArgs& a, hipStream_t stream) {
  conv_shape(a, V);
  hipLaunchKernelGGL((conv_fwd_kernel<CT, W, V>), dim3((unsigned)((long long)a.blocks * a.B * a.groups)), dim3(256), 0, stream,
                     a);
  return check_launch("conv_fwd_kernel");
}
template <typename CT, int W, int V> static int launch_bwd(ConvArgs& a, hipStream_t stream) {
  conv_shape(a, V);
  const long long blocks = (long long)a.blocks * a.B;
  hipLaunchKernelGGL((conv_bwd_kernel<CT, W, V>), dim3((unsigned)(blocks * a.groups)), dim3(256), 0, stream, a);
  const int rc = check_launch("conv_bwd_kernel");
  if (rc) return rc;
  hipLaunchKernelGGL(conv_join_kernel, dim3((unsigned)(((long long)(W + 1) * a.C + 63) / 64)), dim3(256), 0, stream, a,
                     (int)blocks);
  return check_launch("conv_join_kernel");
}
template <typename CT, int W> static int launch_conv(ConvArgs& a, bool bwd, hipStream_t stream) {
  constexpr int F = ConvLanes<CT, W>::FWD, B = ConvLanes<CT, W>::BWD;
  if (bwd) return a.C < B ? launch_bwd<CT, W, 1>(a, stream) : launch_bwd<CT, W, B>(a, stream);
  return a.C < F ? launch_fwd<CT, W, 1>(a, stream) : launch_fwd<CT, W, F>(a, stream);
}

// Tokens a wave takes of a packed row: as many as leave two waves a SIMD.
static int packed_span(const ConvPackedArgs& p, int groups) {
  int span = 32;
  while (span > 8 && (long long)p.N / span * groups < 2048) span /= 2;
  return span;
}
// Workgroups of a packed call, four waves each.
long long conv_packed_groups(const ConvPackedArgs& p) {
  const int lanes = 64 * conv_lanes(1 << 20, p.a.W, p.a.dtype, false), groups = (p.a.C + lanes - 1) / lanes;
  const long long items = p.offsets ? (long long)p.N / packed_span(p, groups) + p.n : p.n;
  return (items + 3) / 4 * groups;
}

template <typename CT, int W> static int launch_packed(ConvPackedArgs& p, hipStream_t stream) {
  constexpr int V = ConvLanes<CT, W>::FWD;
  p.a.groups = (p.a.C + 64 * V - 1) / (64 * V);
  p.a.span = packed_span(p, p.a.groups);
  const dim3 grid((unsigned)conv_packed_groups(p));
  if (p.a.C % V == 0) hipLaunchKernelGGL((conv_packed_kernel<CT, W, V, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((conv_packed_kernel<CT, W, V, false>), grid, dim3(256), 0, stream, p);
  return check_launch("conv_packed_kernel");
}

#define GDNX_CONV_W(CALL)        \
  switch (a_W) {                 \
    case 2: return CALL(2);      \
    case 3: return CALL(3);      \
    case 4: return CALL(4);      \
    case 5: return CALL(5);      \
    case 6: return CALL(6);      \
    case 7: return CALL(7);      \
    default: return CALL(8);     \
  }

int conv_dispatch(ConvArgs& a, bool bwd, hipStream_t stream) {
  const int a_W = a.W;
#define GDNX_CALL_B(w) launch_conv<bf16, w>(a, bwd, stream)
#define GDNX_CALL_F(w) launch_conv<float, w>(a, bwd, stream)
  if (a.dtype == GDNX_DTYPE_BF16) GDNX_CONV_W(GDNX_CALL_B)
  GDNX_CONV_W(GDNX_CALL_F)
#undef GDNX_CALL_B
#undef GDNX_CALL_F
}

int conv_packed_dispatch(ConvPackedArgs& p, hipStream_t stream) {
  const int a_W = p.a.W;
#define GDNX_CALL_B(w) launch_packed<bf16, w>(p, stream)
#define GDNX_CALL_F(w) launch_packed<float, w>(p, stream)
  if (p.a.dtype == GDNX_DTYPE_BF16) GDNX_CONV_W(GDNX_CALL_B)
  GDNX_CONV_W(GDNX_CALL_F)
#undef GDNX_CALL_B
#undef GDNX_CALL_F
}
#undef GDNX_CONV_W

}  // namespace gdnx
