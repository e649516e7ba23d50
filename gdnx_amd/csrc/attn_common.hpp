// What the attention kernels share: the visibility rule and the walk over the
// key tiles that a tile of queries sees.
//
// Query i of Tq stands at position p = i + Tk - Tq.  It sees key j when
//   j <= p,  p < len,  and  p - j < window  or  j < sinks.
// A query outside [0, len) sees nothing: its output and gradients are zero.
#pragma once
#include "gdnx_common.hpp"
#include "gdnx_internal.hpp"

namespace gdnx {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// What rounding to bf16 leaves over (0 where there is no finite rest).
__device__ __forceinline__ float bf16_rest(float x) {
  const float r = x - (float)(bf16)x;
  return fabsf(r) < INFINITY ? r : 0.f;
}

// (p < 0 stands for a query that sees nothing)
__device__ __forceinline__ bool attn_visible(int p, int j, int window, int sinks) {
  return j <= p && (p - j < window || j < sinks);
}

// Whether a query of [off, len) sees key j: its first possible one is the nearest.
__device__ __forceinline__ bool key_seen(int j, int off, int len, int window, int sinks) {
  const int p = max(j, off);
  return p < len && attn_visible(p, j, window, sinks);
}

// Key tiles of BK that queries at positions [p0, p1] see, sinks first: tile
// `it` of `count` starts at key start(it).
template <int BK> struct KeyTiles {
  int n_sink, lo, count;
  __device__ __forceinline__ KeyTiles(int p0, int p1, int len, int window, int sinks) {
    const int hi = min(p1 + 1, len);                       // keys [0, hi)
    if (hi <= 0 || p0 >= len) { n_sink = lo = count = 0; return; }
    const int first = p0 - window + 1 > 0 ? p0 - window + 1 : 0;
    lo = first / BK;
    n_sink = min((sinks + BK - 1) / BK, lo);
    count = n_sink + (hi + BK - 1) / BK - lo;
  }
  __device__ __forceinline__ int start(int it) const { return (it < n_sink ? it : it - n_sink + lo) * BK; }
};

// Query positions [first, end) that see some key of [k0, k0 + BK): those of
// the window, and every later one where the tile holds sinks.
template <int BK> __device__ __forceinline__ int last_query(int k0, int len, int window, int sinks) {
  if (k0 < sinks) return len;
  const long long e = (long long)k0 + BK - 1 + window;
  return e < len ? (int)e : len;
}

// Rows of one key head: (query, head of the group) pairs, heads fastest; row r
// of a tile that starts at row `first`.
struct RowMap {
  int i0, rem, G;
  unsigned magic;       // ceil(2^32 / G): exact for the small numbers of a tile
  __device__ __forceinline__ RowMap(int first, int G_, unsigned magic_) : G(G_), magic(magic_) {
    i0 = first / G;
    rem = first - i0 * G;
  }
  __device__ __forceinline__ void advance(int rows) {
    const int q = div(rem + rows);
    i0 += q;
    rem += rows - q * G;
  }
  __device__ __forceinline__ int div(int x) const { return G == 1 ? x : (int)__umulhi((unsigned)x, magic); }
  __device__ __forceinline__ void at(int r, int* i, int* g) const {
    const int x = r + rem, q = div(x);
    *i = i0 + q;
    *g = x - q * G;
  }
  __device__ __forceinline__ int last(int r) const { return i0 + div(r + rem); }      // the query of row r
};

}  // namespace gdnx
