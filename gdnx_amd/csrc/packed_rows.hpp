// Packed rows: row i of n has tokens offsets[i] .. offsets[i + 1] - 1 of N,
// without padding.  Offsets are clamped to [0, N], so whatever they hold, what
// is found lies within the batch.
#pragma once
#include "gdnx_common.hpp"

namespace gdnx {

__device__ __forceinline__ int packed_offset(const int* offsets, int i, int N) { return min(max(offsets[i], 0), N); }

// The last of [0, n) with f(i) <= x (f does not fall), -1 if there is none: a
// whole wave looks, 64 places a step.
template <typename F> __device__ __forceinline__ int wave_find(int n, long long x, int lane, const F& f) {
  int lo = 0, size = n;
  while (size > 0) {
    const int step = (size + 63) / 64, i = lane * step;
    const int cnt = __popcll(__ballot(i < size && f(lo + i) <= x));
    if (cnt == 0) return -1;
    lo += (cnt - 1) * step;
    if (step == 1) return lo;
    size = min(step, size - (cnt - 1) * step);
  }
  return -1;
}

// x of another lane, 0 where there is none or its row of 16 is not in ROWS.
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ long long dpp(long long x) {
  return (long long)dpp<CTRL, ROWS>((int)(x >> 32)) << 32 | (unsigned)dpp<CTRL, ROWS>((int)x);
}
// Inclusive prefix sum over the wave: within rows of 16, then their last
// lanes' sums to the rows behind.
template <typename T> __device__ __forceinline__ T wave_scan(T x) {
  x += dpp<0x111, 0xf>(x);           // row_shr 1, 2, 4, 8
  x += dpp<0x112, 0xf>(x);
  x += dpp<0x114, 0xf>(x);
  x += dpp<0x118, 0xf>(x);
  x += dpp<0x142, 0xa>(x);           // row_bcast 15, 31
  x += dpp<0x143, 0xc>(x);
  return x;
}

// Rows cut into tiles of T units, a token being G of them: row i owns the work
// items from offsets[i] G / T + i on (floor), which are as many as its tiles at
// least and one for an empty row; N G / T + n items cover every row, whatever
// their lengths, without a plan.  Finds an item's row, its first token and
// their number, and its tile; false: the item is nobody's.  (Uniform in the
// wave; offsets null: one token a row.)
__device__ __forceinline__ bool row_item(const int* offsets, int rows, int N, int G, int T, int item, int lane, int* row,
                                         int* first, int* count, int* tile) {
  if (!offsets) {
    *row = *first = item;
    *count = 1;
    *tile = 0;
    return item < rows;
  }
  const auto at = [&](int i) { return (long long)packed_offset(offsets, i, N) * G / T + i; };
  const int i = wave_find(rows, item, lane, at);
  if (i < 0) return false;
  *row = i;
  *first = packed_offset(offsets, i, N);
  *count = max(packed_offset(offsets, i + 1, N) - *first, 0);
  *tile = item - (int)at(i);
  return *tile >= 0;                 // (offsets that fall may lead anywhere in the batch)
}

}  // namespace gdnx
