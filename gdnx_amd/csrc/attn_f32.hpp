// Tiles in LDS of the float32 attention kernels: 32 rows, D + 4 words apart.
#pragma once
#include "attn_common.hpp"

namespace gdnx {

template <int D> struct F32Tile {
  static constexpr int LD = D + 4, NS = D / 16, BT = 32, WORDS = BT * LD;
};

// Fragment over rows kb .. kb + 15 of a tile, column c of the lane.
template <int LD> __device__ __forceinline__ f32x4 ld_cols(const float* t, int kb, int c, int g) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = t[(kb + 4 * g + i) * LD + c];
  return r;
}

// 32 rows of two matrices by way of registers; a row's places come from
// at(r, &a, &b), which clamps r to a valid row.
template <int D> struct F32Stage {
  static constexpr int UPR = D / 4, N = 32 * UPR / 256, STEP = 256 / UPR;
  f32x4 x[N], y[N];
  int row, unit;
  __device__ __forceinline__ F32Stage(int tid) : row(tid / UPR), unit(tid % UPR) {}
  template <typename At> __device__ __forceinline__ void load(const At& at) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float *pa, *pb;
      at(row + i * STEP, &pa, &pb);
      x[i] = *(const f32x4*)(pa + 4 * unit);
      y[i] = *(const f32x4*)(pb + 4 * unit);
    }
  }
  __device__ __forceinline__ void store(float* ta, float* tb) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = (row + i * STEP) * F32Tile<D>::LD + 4 * unit;
      *(f32x4*)(ta + o) = x[i];
      *(f32x4*)(tb + o) = y[i];
    }
  }
};

}  // namespace gdnx
