// Short causal convolution along a sequence, a filter of W taps for every
// channel, with its activation (gfx950).
//
//   u_t = bias + sum_k w[W-1-k] x_{t-k},   y_t = u_t sigmoid(u_t)  (or u_t)
//   du_t = dy_t s (1 + u_t (1 - s)),  s = sigmoid(u_t);
//   dx_t = sum_k w[W-1-k] du_{t+k},  dw[W-1-k] = sum_t du_t x_{t-k},  dbias = sum_t du_t
//
// x before a sequence's first token is its state, the last W - 1 inputs.
// Channels are contiguous: a lane takes a few of them and walks along the
// tokens with the last W - 1 inputs in registers, so x is read once but for the
// W - 1 rows before each span.  Sums are float32.
//
// Bound by memory and by the vector units, which are busy 63 % of the forward's
// cycles and 66 % of the backward's (26 instructions a value, its exponential
// and reciprocal at a quarter of the rate): 4 x 4096 tokens, 6144 channels, bf16 on four
// taps 75 to 83 us forward (402 MB, 4.8 to 5.4 TB/s; a large copy reaches 5.2) and 141
// backward (604 MB, 4.3 TB/s).  A serving step of 2.4 thousand packed tokens 16 us
// (64 MB), three single tokens 4.8 us.  Behind a row's end a token adds nothing, which
// costs nothing: those of a span that lie before it go without the test.
#include <type_traits>

#include "gdnx_internal.hpp"
#include "packed_rows.hpp"

namespace gdnx {

namespace {

// V channels of a row as they lie in memory; rows may have any alignment.
template <typename CT, int V> struct Raw {
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

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// w[k] multiplies x_{t-k}; filter and bias times log2(e) where there is an
// activation, whose exponential is one of 2.
template <typename WT, int W, int V>
__device__ __forceinline__ void ld_weights(float (*w)[V], float* bias, const ConvArgs& a, int c) {
  WT x[V * W], b[V];
  __builtin_memcpy(x, (const WT*)a.weight + (long long)c * W, sizeof(x));
  if (a.bias) __builtin_memcpy(b, (const WT*)a.bias + c, sizeof(b));
  const float scale = a.silu ? kLog2e : 1.f;
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = to_f(x[e * W + W - 1 - k]) * scale;
    bias[e] = a.bias ? to_f(b[e]) * scale : 0.f;
  }
}
template <int W, int V> __device__ __forceinline__ void ld_weights(float (*w)[V], float* bias, const ConvArgs& a, int c) {
  if (a.wdtype == GDNX_DTYPE_BF16) ld_weights<bf16, W, V>(w, bias, a, c);
  else ld_weights<float, W, V>(w, bias, a, c);
}

// u log2(e) (u without an activation) of a token
template <int W, int V>
__device__ __forceinline__ void conv_sum(float* u, const float (*w)[V], const float* bias, const float (*x)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    u[e] = bias[e];
#pragma unroll
    for (int k = 0; k < W; ++k) u[e] = fmaf(w[k][e], x[k][e], u[e]);
  }
}
// The reciprocals are the hardware's, of one unit in the last place (a
// division takes ten instructions).
template <int W, int V>
__device__ __forceinline__ void conv_out(float* y, const float (*w)[V], const float* bias, const float (*x)[V], int silu) {
  conv_sum<W, V>(y, w, bias, x);
  if (silu) {
#pragma unroll
    for (int e = 0; e < V; ++e)                    // u / (1 + 2^-u), u = y / log2(e)
      y[e] *= __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(-y[e]), kLog2e, kLog2e));
  }
}

// A thread's channels and tokens: lanes of a workgroup side by side on the
// channels, its 256 >> lx_log rows of them on spans of tokens.  Where V does
// not divide C, the last channels are taken twice, by two lanes that store
// the same.  WIDE: a wave is one row of lanes, its tokens and the rows'
// places are scalars.
template <int V, bool WIDE> struct ConvPlace {
  int c, b, t0;
  bool there;
  __device__ __forceinline__ static int channel(const ConvArgs& a, int unit) { return min(unit * V, a.C - V); }
  __device__ __forceinline__ ConvPlace(const ConvArgs& a) {
    const int lx = threadIdx.x & ((1 << a.lx_log) - 1);
    const int ly = WIDE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)threadIdx.x >> a.lx_log;
    int w = blockIdx.x;
    const int g = w % a.groups; w /= a.groups;
    b = w / a.blocks;
    const int unit = (g << a.lx_log) + lx;
    c = channel(a, unit);
    t0 = ((w - b * a.blocks) * (256 >> a.lx_log) + ly) * a.span;
    there = unit * V < a.C && t0 < a.T;
  }
};

// A row's channels: its place and 32 bits of offset.
template <typename CT> __device__ __forceinline__ const CT* chan_at(const CT* row, int c) {
  return (const CT*)((const char*)row + (unsigned)c * (unsigned)sizeof(CT));
}
template <typename CT> __device__ __forceinline__ CT* chan_at(CT* row, int c) {
  return (CT*)((char*)row + (unsigned)c * (unsigned)sizeof(CT));
}

// Rows of a sequence of `len` tokens.  Loads are made whatever t is, from the
// nearest valid token, so that many are in flight; what they give is masked.
template <typename CT, int V> struct ConvRow {
  const CT *x, *state;
  long long xt;
  int len, last, W1, C, c;
  __device__ __forceinline__ ConvRow(const ConvArgs& a, int b, int c_)
      : x((const CT*)a.x + b * a.xs[0]), state(a.state ? (const CT*)a.state + (long long)b * (a.W - 1) * a.C : nullptr),
        xt(a.xs[1]), W1(a.W - 1), C(a.C), c(c_) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    last = max(len - 1, 0);
  }
  __device__ __forceinline__ Raw<CT, V> load(int t) const {
    Raw<CT, V> r;
    r.load(chan_at(x + min(t, last) * xt, c));
    return r;
  }
  // any t < len: the state before token 0, zeros where there is none
  __device__ __forceinline__ void at(float* out, int t) const {
    Raw<CT, V> r;
    if (t >= 0) {
      r.load(chan_at(x + min(t, last) * xt, c));
      r.get(out, len > 0);
    } else if (state) {
      r.load(chan_at(state + (long long)(W1 + t) * C, c));
      r.get(out);
    } else {
      zero_chan<V>(out);
    }
  }
};

}  // namespace

template <typename CT, int W, int V, bool WIDE> __global__ void __launch_bounds__(256) conv_fwd_kernel(ConvArgs a) {
  constexpr int U = 4;
  const ConvPlace<V, WIDE> pl(a);
  if (!pl.there) return;
  const ConvRow<CT, V> row(a, pl.b, pl.c);
  float w[W][V], bias[V], x[W][V];
  Raw<CT, V> next[U];
#pragma unroll
  for (int i = 0; i < U; ++i) next[i] = row.load(pl.t0 + i);
  ld_weights<W, V>(w, bias, a, pl.c);
#pragma unroll
  for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
  const int t1 = min(pl.t0 + a.span, a.T), whole = min(t1, row.len);
  CT* y = (CT*)a.y + ((long long)pl.b * a.T + pl.t0) * a.C;
  for (int t = pl.t0; t < t1; t += U) {
    Raw<CT, V> in[U];
#pragma unroll
    for (int i = 0; i < U; ++i) in[i] = next[i];
#pragma unroll
    for (int i = 0; i < U; ++i) next[i] = row.load(t + U + i);
    const bool all = t + U <= whole;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      shift<W, V>(x);
      in[i].get(x[0]);
      float o[V];
      conv_out<W, V>(o, w, bias, x, a.silu);
      if (!all && t + i >= row.len) zero_chan<V>(o);
      if (all || t + i < t1) st_chan<CT, V>(chan_at(y, pl.c), o);
      y += a.C;
    }
  }
  if (a.state_out && pl.t0 == 0) {           // the last W - 1 inputs before len
    CT* so = (CT*)a.state_out + (long long)pl.b * (W - 1) * a.C;
#pragma unroll
    for (int m = 0; m < W - 1; ++m) {
      float s[V];
      row.at(s, row.len - (W - 1) + m);
      st_chan<CT, V>(chan_at(so + (long long)m * a.C, pl.c), s);
    }
  }
}

// The gradients of a span in one walk along its tokens and the W - 1 behind
// it: du_t goes into the W sums dx_{t-k} that wait for it, the oldest of which
// is then whole.  Filter gradients are summed over the span, then over the
// workgroup, and stored [block][W + 1][C] for the join.
//
// With v = u log2(e) and filters scaled alike, ln 2 du = dy s (ln 2 + v (ln 2)^2 (1 - s))
// makes scaled filters times ln 2 du the plain sum dx, and dw and dbias ln 2 times
// what they are, which is made good once at the end.  The tokens that are all of the span's
// go without a test (with one for each 157 us in the training step above).
template <typename CT, int W, int V, bool WIDE> __global__ void __launch_bounds__(256) conv_bwd_kernel(ConvArgs a) {
  constexpr int U = 4;
  __shared__ float sh[256 * V];
  const ConvPlace<V, WIDE> pl(a);
  float dw[W][V], db[V];
#pragma unroll
  for (int k = 0; k < W; ++k) zero_chan<V>(dw[k]);
  zero_chan<V>(db);
  if (pl.there) {
    const ConvRow<CT, V> row(a, pl.b, pl.c);
    const long long at = (long long)pl.b * a.T * a.C, sat = (long long)pl.b * (W - 1) * a.C;
    const CT* dy = (const CT*)a.dy + at;
    CT* dx = (CT*)a.dx + at;
    float w[W][V], bias[V], x[W][V], acc[W][V];
    Raw<CT, V> nx[U], ng[U];
    const auto ask = [&](int i, int t) {
      nx[i] = row.load(t);
      ng[i].load(chan_at(dy + (long long)min(t, row.last) * a.C, pl.c));
    };
#pragma unroll
    for (int i = 0; i < U; ++i) ask(i, pl.t0 + i);
    ld_weights<W, V>(w, bias, a, pl.c);
#pragma unroll
    for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
#pragma unroll
    for (int k = 0; k < W; ++k) zero_chan<V>(acc[k]);
    const int t1 = min(pl.t0 + a.span, a.T), whole = min(t1, row.len);
    // x of token t into the window, its du into the sums that wait for it
    const auto token = [&](const Raw<CT, V>& rx, const Raw<CT, V>& rg, bool there, bool mine) {
      float du[V];
      shift<W, V>(x);
      shift<W, V>(acc);
      if (there) {
        rx.get(x[0]);
        rg.get(du);
        if (a.silu) {
          float v[V];
          conv_sum<W, V>(v, w, bias, x);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-v[e]));
            du[e] *= s * fmaf(v[e], fmaf(-kLn2 * kLn2, s, kLn2 * kLn2), kLn2);
          }
        }
      } else {                                   // (behind the row: nothing, where 0 times a tap or an input may be NaN)
        zero_chan<V>(x[0]);
        zero_chan<V>(acc[0]);
        return;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        acc[0][e] = w[0][e] * du[e];
#pragma unroll
        for (int k = 1; k < W; ++k) acc[k][e] = fmaf(w[k][e], du[e], acc[k][e]);
      }
      if (mine) {
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k][e] = fmaf(du[e], x[k][e], dw[k][e]);
        if (a.dbias) {
#pragma unroll
          for (int e = 0; e < V; ++e) db[e] += du[e];
        }
      }
    };
    // dx of token tau, which is whole
    const auto put = [&](int tau) {
      if (tau >= t1 || (tau < pl.t0 && pl.t0 > 0)) return;
      const int m = tau - row.len + W - 1;       // its place in the state that is handed on
      if (a.dstate_out && tau < row.len && m >= 0) {
        Raw<CT, V> so;
        float s[V];
        so.load(chan_at((const CT*)a.dstate_out + sat + (long long)m * a.C, pl.c));
        so.get(s);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[W - 1][e] += s[e];
      }
      if (tau >= 0) st_chan_nt<CT, V>(chan_at(dx + (long long)tau * a.C, pl.c), acc[W - 1]);
      else if (a.dstate) st_chan<CT, V>(chan_at((CT*)a.dstate + sat + (long long)(tau + W - 1) * a.C, pl.c), acc[W - 1]);
    };
    int t = pl.t0;
    const auto some = [&](int end) {             // up to `end`, whatever the tokens are
      for (; t < end; t += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          token(nx[i], ng[i], t + i < row.len, t + i < t1);
          put(t + i - (W - 1));
          ask(i, t + U + i);
        }
      }
    };
    some(min(pl.t0 + W - 1, t1));                // dx of these is the span's before, or the state's
    for (; t + U <= whole; t += U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        token(nx[i], ng[i], true, true);
        st_chan_nt<CT, V>(chan_at(dx + (long long)(t + i - (W - 1)) * a.C, pl.c), acc[W - 1]);
        ask(i, t + U + i);
      }
    }
    some(t1 + W - 1);                            // the filter gradients of those behind t1 are the next span's
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
      if (unit * V < a.C) out[(long long)k * a.C + ConvPlace<V, WIDE>::channel(a, unit) + u % V] = s;
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
  s = (sh[0][lane] + sh[1][lane] + sh[2][lane] + sh[3][lane]) * (a.silu ? kLog2e : 1.f);      // (conv_bwd_kernel)
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
// 151 us in the training step of 4 x 4096 tokens and 6144 channels, four 141),
// two in float32 from W = 5 on.
template <typename CT, int W> struct ConvLanes {
  static constexpr int FWD = 16 / sizeof(CT) / (W <= 4 ? 1 : 2), BWD = FWD < 4 ? FWD : 4;
};
static int conv_lanes(int C, int W, int dtype, bool bwd) {
  const int fwd = (dtype == GDNX_DTYPE_BF16 ? 8 : 4) / (W <= 4 ? 1 : 2), V = bwd && fwd > 4 ? 4 : fwd;
  return C < V ? 1 : V;
}

// Lanes on the channels (a power of two up to 64), groups of them, tokens a
// thread takes and blocks of a row: the longest span that gives 1024 workgroups.
// With 512 / 1024 / 2048 of them the forward is the same within 5 %; forward and
// backward of 4 x 4096 tokens, bf16, captured: 1024 channels 45 / 53 / 61 us (the join
// of more blocks), 6144 channels 216 / 215 / 220, smaller calls alike.  Rows of few
// tokens and few channels leave lanes of a workgroup idle (4096 x 64 tokens, 64
// channels: forward 85 us for 67 MB).
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
  const dim3 grid((unsigned)((long long)a.blocks * a.B * a.groups));
  if (V > 1 && a.lx_log == 6) hipLaunchKernelGGL((conv_fwd_kernel<CT, W, V, (V > 1)>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((conv_fwd_kernel<CT, W, V, false>), grid, dim3(256), 0, stream, a);
  return check_launch("conv_fwd_kernel");
}
template <typename CT, int W, int V> static int launch_bwd(ConvArgs& a, hipStream_t stream) {
  conv_shape(a, V);
  const long long blocks = (long long)a.blocks * a.B;
  const dim3 grid((unsigned)(blocks * a.groups));
  if (V > 1 && a.lx_log == 6) hipLaunchKernelGGL((conv_bwd_kernel<CT, W, V, (V > 1)>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((conv_bwd_kernel<CT, W, V, false>), grid, dim3(256), 0, stream, a);
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

// Tokens a wave takes of a packed row: as many as leave two waves a SIMD (2048).
// With 1024 / 2048 / 4096 waves, bf16: 64 x 40 tokens of 6144 channels 17.5 / 17.0 / 17.1
// us, 16 x 500 of 2048 channels 17.0 / 15.6 / 15.6, smaller calls alike.
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
