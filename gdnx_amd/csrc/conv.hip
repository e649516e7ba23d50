// Short causal convolution along a sequence, a filter of W taps for every
// channel, with its activation (gfx950).
//
//   u_t = bias + sum_k w[W-1-k] x_{t-k},   y_t = u_t sigmoid(u_t)  (or u_t)
//   du_t = dy_t s (1 + u_t (1 - s)),  s = sigmoid(u_t);
//   dx_t = sum_k w[W-1-k] du_{t+k},  dw[W-1-k] = sum_t du_t x_{t-k},  dbias = sum_t du_t
//
// x before a sequence's first token is its state, the last W - 1 inputs.
// Channels are contiguous: a lane takes 16 bytes of them (8 from W = 5 on)
// and walks along the tokens with the last W - 1 inputs in registers, so x is
// read once but for the W - 1 rows before each span.  Sums are float32.
#include "gdnx_internal.hpp"
#include "packed_rows.hpp"

namespace gdnx {

namespace {

template <typename CT, int V> struct Vec {
  typedef CT type __attribute__((ext_vector_type(V)));
};

// V channels at p, of which n are there; rows of any alignment.
template <typename CT, int V> __device__ __forceinline__ void ld_chan(float* out, const CT* p, int n) {
  if (n >= V) {
    typename Vec<CT, V>::type x;
    __builtin_memcpy(&x, p, sizeof(x));
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = to_f(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = e < n ? to_f(p[e]) : 0.f;
  }
}
template <typename CT, int V> __device__ __forceinline__ void st_chan(CT* p, const float* in, int n) {
  if (n >= V) {
    typename Vec<CT, V>::type x;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = from_f<CT>(in[e]);
    __builtin_memcpy(p, &x, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) p[e] = from_f<CT>(in[e]);
  }
}
template <int V> __device__ __forceinline__ void zero_chan(float* x) {
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = 0.f;
}
template <int V> __device__ __forceinline__ void copy_chan(float* x, const float* y) {
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = y[e];
}

__device__ __forceinline__ float weight_at(const void* p, long long i, int wdtype) {
  return wdtype == GDNX_DTYPE_BF16 ? to_f(((const bf16*)p)[i]) : ((const float*)p)[i];
}
// w[k] multiplies x_{t-k}
template <int W, int V> __device__ __forceinline__ void ld_weights(float (*w)[V], float* bias, const ConvArgs& a, int c, int nc) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][e] = e < nc ? weight_at(a.weight, (long long)(c + e) * W + W - 1 - k, a.wdtype) : 0.f;
    bias[e] = a.bias && e < nc ? weight_at(a.bias, c + e, a.wdtype) : 0.f;
  }
}

__device__ __forceinline__ float sigmoid(float u) { return 1.f / (1.f + __expf(-u)); }

template <int W, int V>
__device__ __forceinline__ void conv_out(float* y, const float (*w)[V], const float* bias, const float (*x)[V], int silu) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float u = bias[e];
#pragma unroll
    for (int k = 0; k < W; ++k) u = fmaf(w[k][e], x[k][e], u);
    y[e] = silu ? u / (1.f + __expf(-u)) : u;
  }
}

template <int W, int V> __device__ __forceinline__ void shift(float (*x)[V]) {
#pragma unroll
  for (int k = W - 1; k > 0; --k) copy_chan<V>(x[k], x[k - 1]);
}

// A thread's channels and tokens: LX lanes of a workgroup side by side on the
// channels, its 256 / LX rows of them on spans of tokens.
template <int V> struct ConvPlace {
  int c, nc, b, t0;
  __device__ __forceinline__ ConvPlace(const ConvArgs& a) {
    const int lx = threadIdx.x & ((1 << a.lx_log) - 1), ly = threadIdx.x >> a.lx_log;
    int w = blockIdx.x;
    const int g = w % a.groups; w /= a.groups;
    b = w / a.blocks;
    c = ((g << a.lx_log) + lx) * V;
    nc = a.C - c;
    t0 = ((w - b * a.blocks) * (256 >> a.lx_log) + ly) * a.span;
  }
};

// x at token t of a row of `len`: the state before token 0, zeros where there is none.
template <typename CT, int V> struct ConvRow {
  const CT *x, *state;
  long long xt;
  int len, W1, C, nc;
  __device__ __forceinline__ ConvRow(const ConvArgs& a, int b, int c, int nc_)
      : x((const CT*)a.x + b * a.xs[0] + c), state(a.state ? (const CT*)a.state + (long long)b * (a.W - 1) * a.C + c : nullptr),
        xt(a.xs[1]), W1(a.W - 1), C(a.C), nc(nc_) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  }
  __device__ __forceinline__ void at(float* out, int t) const {
    if (t >= 0 && t < len) ld_chan<CT, V>(out, x + t * xt, nc);
    else if (t < 0 && state) ld_chan<CT, V>(out, state + (long long)(W1 + t) * C, nc);
    else zero_chan<V>(out);
  }
};

}  // namespace

template <typename CT, int W, int V> __global__ void __launch_bounds__(256) conv_fwd_kernel(ConvArgs a) {
  constexpr int U = 8;
  const ConvPlace<V> pl(a);
  if (pl.nc <= 0 || pl.t0 >= a.T) return;
  const ConvRow<CT, V> row(a, pl.b, pl.c, pl.nc);
  float w[W][V], bias[V], x[W][V];
  ld_weights<W, V>(w, bias, a, pl.c, pl.nc);
#pragma unroll
  for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
  const int t1 = min(pl.t0 + a.span, a.T);
  CT* y = (CT*)a.y + ((long long)pl.b * a.T + pl.t0) * a.C + pl.c;
  for (int t = pl.t0; t < t1; t += U) {
    float in[U][V];
#pragma unroll
    for (int i = 0; i < U; ++i) row.at(in[i], t + i);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      shift<W, V>(x);
      copy_chan<V>(x[0], in[i]);
      float o[V];
      conv_out<W, V>(o, w, bias, x, a.silu);
      if (t + i >= row.len) zero_chan<V>(o);
      if (t + i < t1) st_chan<CT, V>(y, o, pl.nc);
      y += a.C;
    }
  }
  if (a.state_out && pl.t0 == 0) {           // the last W - 1 inputs before len
    CT* so = (CT*)a.state_out + (long long)pl.b * (W - 1) * a.C + pl.c;
#pragma unroll
    for (int m = 0; m < W - 1; ++m) {
      float s[V];
      row.at(s, row.len - (W - 1) + m);
      st_chan<CT, V>(so + (long long)m * a.C, s, pl.nc);
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
  if (pl.nc > 0 && pl.t0 < a.T) {
    const ConvRow<CT, V> row(a, pl.b, pl.c, pl.nc);
    float w[W][V], bias[V], x[W][V], acc[W][V];
    ld_weights<W, V>(w, bias, a, pl.c, pl.nc);
#pragma unroll
    for (int k = 1; k < W; ++k) row.at(x[k - 1], pl.t0 - k);
#pragma unroll
    for (int k = 0; k < W; ++k) zero_chan<V>(acc[k]);
    const int t1 = min(pl.t0 + a.span, a.T);
    const long long at = (long long)pl.b * a.T * a.C + pl.c;
    const CT* dy = (const CT*)a.dy + at;
    CT* dx = (CT*)a.dx + at;
    const long long sat = (long long)pl.b * (W - 1) * a.C + pl.c;
    for (int t = pl.t0; t < t1 + W - 1; t += U) {
      float in[U][V], g[U][V];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        row.at(in[i], t + i);
        if (t + i < row.len) ld_chan<CT, V>(g[i], dy + (long long)(t + i) * a.C, pl.nc);
        else zero_chan<V>(g[i]);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        shift<W, V>(x);
        shift<W, V>(acc);
        copy_chan<V>(x[0], in[i]);
        zero_chan<V>(acc[0]);
        const bool mine = t + i < t1, there = t + i < row.len;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float du = g[i][e];
          if (a.silu) {
            float u = bias[e];
#pragma unroll
            for (int k = 0; k < W; ++k) u = fmaf(w[k][e], x[k][e], u);
            const float s = sigmoid(u);
            du *= s * fmaf(u, 1.f - s, 1.f);
          }
          if (!there) du = 0.f;
#pragma unroll
          for (int k = 0; k < W; ++k) {
            acc[k][e] = fmaf(w[k][e], du, acc[k][e]);
            if (mine) dw[k][e] = fmaf(du, x[k][e], dw[k][e]);
          }
          if (mine) db[e] += du;
        }
        const int tau = t + i - (W - 1);           // dx of this token is whole
        const int m = tau - row.len + W - 1;       // its place in the state that is handed on
        if (tau >= t1 || (tau < pl.t0 && pl.t0 > 0)) continue;
        if (a.dstate_out && tau < row.len && m >= 0) {
          float so[V];
          ld_chan<CT, V>(so, (const CT*)a.dstate_out + sat + (long long)m * a.C, pl.nc);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[W - 1][e] += so[e];
        }
        if (tau >= 0) st_chan<CT, V>(dx + (long long)tau * a.C, acc[W - 1], pl.nc);
        else if (a.dstate) st_chan<CT, V>((CT*)a.dstate + sat + (long long)(tau + W - 1) * a.C, acc[W - 1], pl.nc);
      }
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
      const int c = ((blockIdx.x % a.groups) << a.lx_log) * V + u;
      float s = 0.f;
      for (int r = 0; r < rows; ++r) s += sh[(r << a.lx_log) * V + u];
      if (c < a.C) out[(long long)k * a.C + c] = s;
    }
    __syncthreads();
  }
}

// Blocks' filter gradients summed in order: [blocks][W + 1][C] -> dweight [C,W], dbias [C].
__global__ void __launch_bounds__(256) conv_join_kernel(ConvArgs a, int blocks) {
  const long long u = (long long)blockIdx.x * 256 + threadIdx.x, n = (long long)(a.W + 1) * a.C;
  if (u >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < blocks; ++i) s += a.part[i * n + u];
  const int k = (int)(u / a.C), c = (int)(u % a.C);
  void* to = k < a.W ? a.dweight : a.dbias;
  if (!to) return;
  const long long at = k < a.W ? (long long)c * a.W + a.W - 1 - k : c;
  if (a.wdtype == GDNX_DTYPE_BF16) ((bf16*)to)[at] = (bf16)s;
  else ((float*)to)[at] = s;
}

// Packed rows of unlike lengths, each with a slot of the state pool: a wave
// takes a span of one row's tokens (row_item).  The row's first wave alone
// reads the old state, before it writes the new one.
template <typename CT, int W, int V> __global__ void __launch_bounds__(256) conv_packed_kernel(ConvPackedArgs p) {
  const ConvArgs& a = p.a;
  const int lane = threadIdx.x & 63;
  const int item = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / a.groups) * 4 + (threadIdx.x >> 6));
  const int c = ((int)(blockIdx.x % a.groups) * 64 + lane) * V, nc = a.C - c;
  int i, o0, n, tile;
  if (!row_item(p.offsets, p.n, p.N, 1, a.span, item, lane, &i, &o0, &n, &tile)) return;
  const int t0 = tile * a.span;
  if (nc <= 0 || (t0 >= n && tile > 0)) return;
  const int slot = p.slots ? p.slots[i] : i, to = p.to_slots ? p.to_slots[i] : slot;
  const bool live = slot >= 0 && slot < p.n_slots;
  const CT* x = (const CT*)a.x + o0 * a.xs[1] + c;
  const CT* state = (const CT*)a.state + (long long)(live ? slot : 0) * (W - 1) * a.C + c;
  const auto at = [&](float* out, int t) {
    if (!live || t >= n) zero_chan<V>(out);
    else if (t >= 0) ld_chan<CT, V>(out, x + t * a.xs[1], nc);
    else ld_chan<CT, V>(out, state + (long long)(W - 1 + t) * a.C, nc);
  };
  float w[W][V], bias[V], xw[W][V], next[W - 1][V];
  ld_weights<W, V>(w, bias, a, c, nc);
#pragma unroll
  for (int k = 1; k < W; ++k) at(xw[k - 1], t0 - k);
  if (tile == 0) {
#pragma unroll
    for (int m = 0; m < W - 1; ++m) at(next[m], n - (W - 1) + m);
    if (live && to >= 0 && to < p.n_slots) {
      CT* so = (CT*)a.state_out + (long long)to * (W - 1) * a.C + c;
#pragma unroll
      for (int m = 0; m < W - 1; ++m) st_chan<CT, V>(so + (long long)m * a.C, next[m], nc);
    }
  }
  const int t1 = min(t0 + a.span, n);
  CT* y = (CT*)a.y + ((long long)o0 + t0) * a.C + c;
  for (int t = t0; t < t1; ++t) {
    shift<W, V>(xw);
    at(xw[0], t);
    float o[V];
    conv_out<W, V>(o, w, bias, xw, a.silu);
    if (!live) zero_chan<V>(o);
    st_chan<CT, V>(y, o, nc);
    y += a.C;
  }
}

static int conv_lanes(int W, int dtype) { return (dtype == GDNX_DTYPE_BF16 ? 8 : 4) / (W <= 4 ? 1 : 2); }

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

static ConvArgs shaped(int B, int T, int C, int W, int dtype) {
  ConvArgs a{};
  a.B = B; a.T = T; a.C = C; a.W = W;
  conv_shape(a, conv_lanes(W, dtype));
  return a;
}
long long conv_bwd_blocks(int B, int T, int C, int W, int dtype) { return (long long)shaped(B, T, C, W, dtype).blocks * B; }
long long conv_groups(int B, int T, int C, int W, int dtype) {
  const ConvArgs a = shaped(B, T, C, W, dtype);
  return (long long)a.blocks * B * a.groups;
}

template <typename CT, int W> static int launch_conv(ConvArgs& a, bool bwd, hipStream_t stream) {
  constexpr int V = 16 / sizeof(CT) / (W <= 4 ? 1 : 2);
  conv_shape(a, V);
  const long long blocks = (long long)a.blocks * a.B;
  if (!bwd) {
    hipLaunchKernelGGL((conv_fwd_kernel<CT, W, V>), dim3((unsigned)(blocks * a.groups)), dim3(256), 0, stream, a);
    return check_launch("conv_fwd_kernel");
  }
  hipLaunchKernelGGL((conv_bwd_kernel<CT, W, V>), dim3((unsigned)(blocks * a.groups)), dim3(256), 0, stream, a);
  const int rc = check_launch("conv_bwd_kernel");
  if (rc || (!a.dweight && !a.dbias)) return rc;
  hipLaunchKernelGGL(conv_join_kernel, dim3((unsigned)(((long long)(W + 1) * a.C + 255) / 256)), dim3(256), 0, stream, a,
                     (int)blocks);
  return check_launch("conv_join_kernel");
}

// Workgroups of a packed call, four waves each.
constexpr int kPackedSpan = 8;
long long conv_packed_groups(const ConvPackedArgs& p) {
  const int lanes = 64 * conv_lanes(p.a.W, p.a.dtype);
  const long long items = p.offsets ? (long long)p.N / kPackedSpan + p.n : p.n;
  return (items + 3) / 4 * ((p.a.C + lanes - 1) / lanes);
}

template <typename CT, int W> static int launch_packed(ConvPackedArgs& p, hipStream_t stream) {
  constexpr int V = 16 / sizeof(CT) / (W <= 4 ? 1 : 2);
  p.a.groups = (p.a.C + 64 * V - 1) / (64 * V);
  p.a.span = kPackedSpan;
  hipLaunchKernelGGL((conv_packed_kernel<CT, W, V>), dim3((unsigned)conv_packed_groups(p)), dim3(256), 0, stream, p);
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
