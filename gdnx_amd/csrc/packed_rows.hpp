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
