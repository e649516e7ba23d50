// Attention of one new token over a paged key-value cache (gfx950).
//
// Row s's token stands at position len - 1 of its table row; it sees the last
// `window` tokens and the first `sinks` ones.  The visible keys are counted
// through without a gap, x = 0 .. nvis - 1 (the sinks, then the window), so a
// tile of keys needs no mask but its end.
//
// Bound by HBM: each visible key and value is read once.  256 rows of up to
// 8192 tokens (16 query heads on 4, d = 128, bf16; 2.18 GB) take 400 us,
// 5.4 TB/s; two rows of 262143 tokens (32 on 8; 1.5 GB) 263 us with the join,
// 5.8 TB/s; a large copy reaches 5.1.  A workgroup takes a
// span of one row's keys for one key head and up to 16 of its query heads
// (grouped heads share what is read); its four waves take the span's tiles
// (32 keys in bf16, 16 in float32) in turn, each with its own running
// maximum, sum and output.  A wave's loads go straight to registers, 16 bytes
// a lane and a tile ahead: K rows as MFMA operands, V rows by way of the
// wave's own LDS, read back transposed.  Keys without a page, and those past
// the end, are read from a row of zeros and masked, so nothing that a page
// holds beyond the row's length enters a product.
//
// S^T = K Q^T puts a query head in a lane column: its statistics are in-lane
// maxima and two shuffles, and its probabilities are the operand of
// O^T = V^T P^T: in bf16 they are two, the rounded value and what that leaves
// over, since the matrix units wait for memory anyway (256 rows 384 us with one
// operand and with two; y is 1.7e-3 from 64 bits, which is its own rounding,
// instead of 2.2e-3).  Spans are joined by a second kernel, in order.
#include "attn_paged.hpp"

namespace gdnx {

namespace {
struct Seen {                                     // a row's visible keys
  int len, lo, ns, nvis;
  bool fits;                                      // whether the table has a place for the last token
  __device__ __forceinline__ Seen(const PagedAttnArgs& a, int r) {
    const long long cap = (long long)a.width << a.page_log;
    len = r >= 0 && r < a.rows ? a.lengths[r] : 0;
    fits = len <= cap;
    len = len < 0 ? 0 : len > cap ? (int)cap : len;
    lo = len > a.window ? len - a.window : 0;
    ns = min(a.sinks, lo);
    nvis = ns + len - lo;
  }
};

// spans that a row of n key tiles is cut into: about four tiles each, or more (five
// tiles are cut into three and two)
__device__ __forceinline__ int spans(int tiles, int max_spans) { return min(max_spans, (tiles + 3) / 4); }

}  // namespace

template <typename CT, int D>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PagedAttnArgs a) {
  typedef typename FragT<CT>::type Frag;
  constexpr int BT = FragT<CT>::KSTEP, NU = FragT<CT>::TPS;       // keys a tile, 16-key subtiles
  constexpr int EPU = 16 / sizeof(CT), UPR = D / EPU, NKS = D / FragT<CT>::KSTEP, NT = D / 16;
  constexpr int NV = BT * UPR / 64;                               // 16-byte units of a V tile a lane
  constexpr int STAGE = BT * D * sizeof(CT), OUT = 16 * D * sizeof(float);
  __shared__ __attribute__((aligned(16))) char smem[4 * (STAGE > OUT ? STAGE : OUT)];
  __shared__ long long s_off[4][BT];
  __shared__ float s_m[4][16], s_l[4][16];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, gb = (G + 15) / 16;
  int w = blockIdx.x;
  const int span = w % a.spans; w /= a.spans;
  const int gblk = w % gb; w /= gb;
  const int hk = w % a.Hkv, s = w / a.Hkv;
  const int r = a.slots ? a.slots[s] : s;
  const Seen see(a, r);
  const int tiles = (see.nvis + BT - 1) / BT, parts = spans(tiles, a.spans);
  const int rows = min(16, G - 16 * gblk), h0 = hk * G + 16 * gblk;
  if (span >= parts) {
    if (span == 0)                                                // an empty row
      for (int u = tid; u < rows * (D / 4); u += 256)
        st4((CT*)a.y + ((long long)s * a.Hq + h0) * D + 4 * u, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const int* table = a.table + (long long)r * a.width;
  const long long rowb = D * (int)sizeof(CT), headb = rowb << a.page_log;
  // a new token without a place in the cache is neither written nor seen
  const char* knew = a.k && see.fits ? (const char*)a.k + ((long long)s * a.Hkv + hk) * rowb : nullptr;
  const char* vnew = a.v && see.fits ? (const char*)a.v + ((long long)s * a.Hkv + hk) * rowb : nullptr;
  // the new token goes to its page (nobody reads it there in this call)
  if (knew && span == 0 && gblk == 0 && tid < 2 * UPR) {
    const int pos = see.len - 1, pg = table[pos >> a.page_log], u = tid % UPR;
    if (pg >= 0 && pg < a.n_pages) {
      char* to = (char*)(tid < UPR ? a.k_pages : a.v_pages) + ((long long)pg * a.Hkv + hk) * headb +
                 (pos & ((1 << a.page_log) - 1)) * rowb;
      *(uint4*)(to + 16 * u) = *(const uint4*)((tid < UPR ? knew : vnew) + 16 * u);
    }
  }
  const int per = (tiles + parts - 1) / parts, t0 = span * per, t1 = min(tiles, t0 + per);

  Frag qf[NKS];
#pragma unroll
  for (int c = 0; c < NKS; ++c) {
    if (n < rows) qf[c] = *(const Frag*)((const CT*)a.q + ((long long)s * a.Hq + h0 + n) * D + (4 * c + g) * EPU);
    else qf[c] = Frag{};
  }
  // key x of the visible ones: its page
  const auto page_of = [&](int x) {
    if (x >= see.nvis) return -1;
    const int j = x < see.ns ? x : x - see.ns + see.lo;
    return table[j >> a.page_log];
  };
  Frag kr[NU][NKS];
  u32x4 vr[NV];
  bool live[NU];                       // whether the lane's keys of the tile are visible
  long long* off = s_off[wave];
  CT* stage = (CT*)(smem + wave * STAGE);
  // a tile's rows: lane l < BT finds key l's place (-1: none, -2: the new token)
  const auto load = [&](int t, int pg) {
    wave_lds_sync();
    if (lane < BT) {
      const int x = t * BT + lane, j = x < see.ns ? x : x - see.ns + see.lo;
      long long o = -1;
      if (x < see.nvis && pg >= 0 && pg < a.n_pages)
        o = knew && x == see.nvis - 1 ? -2 : ((long long)pg * a.Hkv + hk) * headb + (j & ((1 << a.page_log) - 1)) * rowb;
      off[lane] = o;
    }
    wave_lds_sync();
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const long long o = off[16 * u + n];
      const GlobalBytes p = (GlobalBytes)(o >= 0 ? (const char*)a.k_pages + o : o == -2 ? knew : (const char*)g_zero_row);
      live[u] = o != -1;
#pragma unroll
      for (int c = 0; c < NKS; ++c) kr[u][c] = ld_global<Frag>(p + (4 * c + g) * 16);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int U = i * 64 + lane, row = U / UPR, u = (U % UPR) ^ v_swizzle<D>((const CT*)nullptr, row);
      const long long o = off[row];
      const GlobalBytes p = (GlobalBytes)(o >= 0 ? (const char*)a.v_pages + o : o == -2 ? vnew : (const char*)g_zero_row);
      vr[i] = ld_global<u32x4>(p + u * 16);
    }
  };

  const float sc = a.scale * kLog2e;
  f32x4 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = zero4();
  float m = -INFINITY, l = 0.f;
  int t = t0 + wave;
  if (t < t1) load(t, lane < BT ? page_of(t * BT + lane) : -1);
  int pg = t + 4 < t1 && lane < BT ? page_of((t + 4) * BT + lane) : -1;
  for (; t < t1; t += 4) {
    f32x4 sx[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      sx[u] = zero4();
#pragma unroll
      for (int c = 0; c < NKS; ++c) mma(sx[u], kr[u][c], qf[c]);
    }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < NV; ++i) *(u32x4*)((char*)stage + (i * 64 + lane) * 16) = vr[i];
    // which keys of the lane's accumulator rows are visible: lane 4 g + e has key 16 u + 4 g + e
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const unsigned long long lv = __ballot(live[u]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sx[u][e] = (lv >> (4 * g + e) & 1) ? sx[u][e] * sc : -INFINITY;
    }
    if (t + 4 < t1) {
      load(t + 4, pg);
      pg = t + 8 < t1 && lane < BT ? page_of((t + 8) * BT + lane) : -1;
    }
    float mx = sx[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sx[u][e]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ms);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sx[u][e] = __builtin_amdgcn_exp2f(sx[u][e] - ms);
        sum += sx[u][e];
      }
    l = l * f + sum;
    m = mn;
    const Frag pf = acc_frag((CT*)nullptr, sx[0], sx[NU - 1]);
    Frag pr{};                           // what rounding P to bf16 leaves over
    if constexpr (sizeof(CT) == 2) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sx[u][e] = bf16_rest(sx[u][e]);
      pr = acc_frag((CT*)nullptr, sx[0], sx[NU - 1]);
    }
    wave_lds_sync();
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      o[c] *= f;
      const Frag vf = v_frag<D>(stage, c, n, g);
      mma(o[c], vf, pf);
      if constexpr (sizeof(CT) == 2) mma(o[c], vf, pr);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the four waves joined
  if (g == 0) {
    s_m[wave][n] = m;
    s_l[wave][n] = l;
  }
  __syncthreads();
  float* so = (float*)smem;
#pragma unroll
  for (int c = 0; c < NT; ++c) *(f32x4*)&so[(wave * 16 + n) * D + 16 * c + 4 * g] = o[c];
  __syncthreads();
  for (int u = tid; u < rows * (D / 4); u += 256) {
    const int q = u / (D / 4), d = 4 * (u % (D / 4));
    float mm = s_m[0][q];
#pragma unroll
    for (int v = 1; v < 4; ++v) mm = fmaxf(mm, s_m[v][q]);
    const float ms = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    f32x4 acc = zero4();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = __builtin_amdgcn_exp2f(s_m[v][q] - ms);
      ll += s_l[v][q] * f;
      acc += *(const f32x4*)&so[(v * 16 + q) * D + d] * f;
    }
    const long long head = (long long)s * a.Hq + h0 + q;
    if (parts == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      st4((CT*)a.y + head * D + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      const long long slot = head * a.spans + span;
      *(f32x4*)(a.part + slot * D + d) = acc;
      if (d == 0) {
        float* ml = a.part + (long long)a.NS * a.Hq * a.spans * D + 2 * slot;
        ml[0] = mm;
        ml[1] = ll;
      }
    }
  }
}

// A workgroup a query head: D / 4 threads take a span's four columns each, the
// groups of them every n-th span, and are joined in order.  (A workgroup a row
// took 20 us for two rows of 128 spans and 32 heads, this form 7.)
template <typename CT, int D> __global__ void __launch_bounds__(256) paged_join_kernel(PagedAttnArgs a) {
  constexpr int BT = FragT<CT>::KSTEP, V = D / 4, NG = 256 / V;
  __shared__ __attribute__((aligned(16))) float s_acc[NG][D];
  __shared__ float s_m[NG], s_l[NG];
  const long long head = blockIdx.x;
  const int s = (int)(head / a.Hq), grp = threadIdx.x / V, d = 4 * (threadIdx.x % V);
  const Seen see(a, a.slots ? a.slots[s] : s);
  const int parts = spans((see.nvis + BT - 1) / BT, a.spans);
  if (parts <= 1) return;                          // written by its workgroup
  const float* ml = a.part + (long long)a.NS * a.Hq * a.spans * D + 2 * head * a.spans;
  const float* po = a.part + head * a.spans * D + d;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = zero4();
  const auto add = [&](float m2, float l2, const f32x4& x) {
    const float mn = fmaxf(m, m2), ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ms), g = __builtin_amdgcn_exp2f(m2 - ms);
    l = l * f + l2 * g;
    acc = acc * f + x * g;
    m = mn;
  };
#pragma unroll 4
  for (int i = grp; i < parts; i += NG) add(ml[2 * i], ml[2 * i + 1], *(const f32x4*)(po + (long long)i * D));
  *(f32x4*)&s_acc[grp][d] = acc;
  if (d == 0) {
    s_m[grp] = m;
    s_l[grp] = l;
  }
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int g = 1; g < NG; ++g) add(s_m[g], s_l[g], *(const f32x4*)&s_acc[g][d]);
  acc *= l == 0.f ? 0.f : 1.f / l;
  st4((CT*)a.y + head * D + d, acc[0], acc[1], acc[2], acc[3]);
}

// Spans of a row of `keys` visible keys.  Two workgroups a CU where the rows
// and heads alone do not give them, each span about four tiles or more; up to six a
// CU (so that rows of unequal lengths level out) while a span keeps 32 tiles,
// beside which a workgroup's start and its share of the join are small.  In us,
// one span / this rule / eight a CU with at least four tiles each:
//   256 rows up to 8192 tokens, 16/4 heads, d = 128    431 / 400 / 400
//   2 rows of 262143 tokens, 32/8, d = 128            2937 / 263 / 268
//   16 rows, window 4096, 16/4, d = 128                 61 /  26 /  35
//   48 rows, window 512, 16/16, d = 64                  19 /  19 /  24
int paged_attn_spans(int NS, int Hq, int Hkv, long long keys, int dtype) {
  const int G = Hq / Hkv, tile = dtype == GDNX_DTYPE_BF16 ? 32 : 16;
  const long long base = (long long)NS * Hkv * ((G + 15) / 16);
  long long n = (512 + base - 1) / base, more = (1536 + base - 1) / base;
  const long long most = (keys + 4 * tile - 1) / (4 * tile);
  if (n > most) n = most;
  if (more > keys / (32 * tile)) more = keys / (32 * tile);
  if (n < more) n = more;
  if (n > 256) n = 256;
  return n < 1 ? 1 : (int)n;
}

template <typename CT, int D> static int launch_paged(const PagedAttnArgs& a, hipStream_t stream) {
  const int G = a.Hq / a.Hkv;
  hipLaunchKernelGGL((paged_attn_kernel<CT, D>), dim3((unsigned)((long long)a.NS * a.Hkv * ((G + 15) / 16) * a.spans)),
                     dim3(256), 0, stream, a);
  int rc = check_launch("paged_attn_kernel");
  if (rc || a.spans == 1) return rc;
  hipLaunchKernelGGL((paged_join_kernel<CT, D>), dim3((unsigned)((long long)a.NS * a.Hq)), dim3(256), 0, stream, a);
  return check_launch("paged_join_kernel");
}

int paged_attn_dispatch(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.dtype == GDNX_DTYPE_BF16)
    return a.D == 128 ? launch_paged<bf16, 128>(a, stream) : launch_paged<bf16, 64>(a, stream);
  return a.D == 128 ? launch_paged<float, 128>(a, stream) : launch_paged<float, 64>(a, stream);
}

}  // namespace gdnx
