// Tiles in LDS and 32 x 32 x 16 matrix operands of the bf16 attention kernels.
//
// v_mfma_f32_32x32x16_bf16, lane l = 32 h + n (checked on gfx950):
//   A: lane supplies A[m = n][k in set(h)], B: B[k in set(h)][n], 8 values;
//   D: element e of the lane is D[8 (e / 4) + 4 h + e % 4][n].
// The k set of a lane is the same permutation for A and B.  Operands whose k
// runs along a row take 8 contiguous values (8 h + i); those contracted over
// accumulator rows take the rows 16 c + 4 h + {0..3} and + 8, as the
// accumulators hold them, read transposed from row-major tiles
// (ds_read_b64_tr_b16: 16 lanes give 4 rows of 16 columns, a lane gets a
// column of 4).
//
// A tile row is D values; its 16-byte units are permuted by an xor with the
// row's bits, so that both reads are free of bank conflicts: 16 rows of one
// unit fall into different units, and 4 rows of 4 units into different
// quarters.
#pragma once
#include "attn_common.hpp"

namespace gdnx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void mma32(f32x16& acc, const bf16x8& a, const bf16x8& b) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
  return (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}
// Rows 16 c .. 16 c + 15 of an accumulator tile as an operand over them.
__device__ __forceinline__ bf16x8 acc_frag32(const f32x16& s, int c) {
  return (bf16x8){(bf16)s[8 * c], (bf16)s[8 * c + 1], (bf16)s[8 * c + 2], (bf16)s[8 * c + 3],
                  (bf16)s[8 * c + 4], (bf16)s[8 * c + 5], (bf16)s[8 * c + 6], (bf16)s[8 * c + 7]};
}
// Maximum / sum over the lanes n and n + 32.
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D> struct Tile {
  static constexpr int RB = 2 * D, UPR = D / 8;      // bytes and 16-byte units of a row
  static constexpr int NS = D / 16, ND = D / 32;     // k steps along a row, 32-column blocks
  __device__ static __forceinline__ int swz(int r) {
    return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  }
  __device__ static __forceinline__ int at(int r, int unit) { return r * RB + ((unit ^ swz(r)) << 4); }
};

// A lane's places in a tile of 32 rows.
template <int D> struct LaneMap {
  using T = Tile<D>;
  int row0, rsw, col0, n, h;
  __device__ __forceinline__ LaneMap(int lane) {
    n = lane & 31;
    h = lane >> 5;
    row0 = n * T::RB;
    rsw = (T::swz(n) ^ h) << 4;
    const int i = lane & 15, c2 = (lane >> 4) & 1;
    col0 = T::at(4 * h + (i >> 2), 2 * c2 + ((i & 3) >> 1)) + 8 * (i & 1);
  }
  // the same places as numbers that the compiler takes for new ones: what is
  // derived from them is not kept in registers from one step to the next
  __device__ __forceinline__ LaneMap fresh() const {
    LaneMap m = *this;
    m.row0 = opaque(row0);
    m.rsw = opaque(rsw);
    m.col0 = opaque(col0);
    return m;
  }
  // row n, k step c
  __device__ __forceinline__ bf16x8 row(const char* tile, int c) const {
    return *(const bf16x8*)(tile + row0 + ((c << 5) ^ rsw));
  }
  // columns 32 t + n over the 16 rows that start at `tile`
  __device__ __forceinline__ bf16x8 cols(const char* tile, int t) const {
    typedef __attribute__((address_space(3))) bf16x4 Lds4;
    // (eight rows on, the units' permutation differs in bit 1)
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds4*)(tile + (col0 ^ (64 * t))));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds4*)(tile + 8 * T::RB + (col0 ^ (64 * t) ^ 32)));
    return (bf16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
  // a transposed accumulator [D][32 rows], times f, as 32 rows of bf16; low:
  // what that rounding leaves over
  __device__ __forceinline__ void put(char* tile, const f32x16* o, float f, bool low = false) const {
#pragma unroll
    for (int t = 0; t < T::ND; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = o[t][4 * i + e] * f;
          if (low) x[e] = bf16_rest(x[e]);
        }
        st4((bf16*)(tile + T::at(n, 4 * t + i) + 8 * h), x[0], x[1], x[2], x[3]);
      }
  }
};

// 64-row tiles of two matrices straight into LDS, 256 threads, 16 bytes a lane:
// an instruction fills 1 KB in lane order, so the units' permutation is made by
// what each lane reads.  Rows beyond the last valid one are read from it (what
// they give is masked).  Offsets within a tile are 32-bit: token strides stay
// below 2^24 elements.
template <int D> struct TileLoad {
  using T = Tile<D>;
  static constexpr int N = 64 * T::UPR / 256, STEP = 256 / T::UPR;
  unsigned row, sa, sb, u;
  int wave;
  __device__ __forceinline__ TileLoad(int tid, int wave_, int as, int bs) : row(tid / T::UPR), wave(wave_) {
    u = ((tid % T::UPR) ^ T::swz(row)) * 16;
    sa = 2 * as;
    sb = 2 * bs;
  }
  __device__ __forceinline__ void load(char* ta, const bf16* a, char* tb, const bf16* b, int last) const {
    typedef __attribute__((address_space(1))) void* G;
    typedef __attribute__((address_space(3))) void* L;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned r = min((int)row + i * STEP, last);
      __builtin_amdgcn_global_load_lds((G)((const char*)a + (r * sa + u)), (L)(ta + i * 4096 + wave * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((G)((const char*)b + (r * sb + u)), (L)(tb + i * 4096 + wave * 1024), 16, 0, 0);
    }
  }
};
// A workgroup barrier after which every wave's loads into LDS are there.  The
// wait (vmcnt 0, lgkmcnt 0) is the builtin, which the compiler counts: it then
// adds none of its own before the tiles are read.
__device__ __forceinline__ void loads_done_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace gdnx
