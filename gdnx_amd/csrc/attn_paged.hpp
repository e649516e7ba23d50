// Reading a page cache's rows as matrix operands: the served step's tiles and
// the short rows of a packed batch.
#pragma once
#include "attn_common.hpp"

namespace gdnx {
namespace {

__device__ const uint4 g_zero_row[32] = {};       // one row of zeros: 512 bytes


// (a choice between pointers is read as memory of any kind, LDS included,
// unless it is said to be global: its loads would then wait for LDS too)
typedef const __attribute__((address_space(1))) char* GlobalBytes;
template <typename V> __device__ __forceinline__ V ld_global(GlobalBytes p) {
  return *(const __attribute__((address_space(1))) V*)p;
}

typedef __bf16 LdsB4 __attribute__((ext_vector_type(4)));

// V^T operand of a 16-wide column block: the lane's column 16 t + n, its keys
// as the score tiles hold them.
template <int D> __device__ __forceinline__ bf16x8 v_frag(const bf16* t, int ct, int n, int g) {
  constexpr int UPR = D / 8;
  bf16x4 x[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = 16 * u + 4 * g + (n >> 2);
    const int sw = UPR == 16 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
    const int unit = (2 * ct + ((n >> 1) & 1)) ^ sw;
    x[u] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) LdsB4*)(t + r * D + unit * 8 + 4 * (n & 1)));
  }
  return (bf16x8){x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
}
template <int D> __device__ __forceinline__ f32x4 v_frag(const float* t, int ct, int n, int g) {
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = 4 * g + e, unit = (4 * ct + (n >> 2)) ^ (4 * ((r >> 2) & 3));
    x[e] = t[r * D + unit * 4 + (n & 3)];
  }
  return x;
}
template <int D> __device__ __forceinline__ int v_swizzle(const bf16*, int r) {
  return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
}
template <int D> __device__ __forceinline__ int v_swizzle(const float*, int r) { return 4 * ((r >> 2) & 3); }

}  // namespace
}  // namespace gdnx
