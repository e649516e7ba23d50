// Windowed attention with sinks for bf16 (gfx950): forward.  Forms and rules
// as in attn_win.hip, on the 32 x 32 x 16 matrix instruction.
#include "attn_spans.hpp"
#include "attn_tiles.hpp"

namespace gdnx {

// Forward.  A workgroup of four waves takes 128 rows of one key head, a row
// being a (query, query head of the group) pair with the heads fastest, so
// that grouped heads share the key tiles and the tile's queries span few
// positions; a wave owns 32 rows.  Key tiles of 64 go straight into LDS,
// double-buffered, one barrier a tile (by way of registers: 1260 instead of
// 1170 thousand cycles for the prompt below).
//   S^T = K Q^T   a lane holds 32 scores of one row
//   O^T += V^T P^T   the score accumulators, as bf16, are the operand (their rest
//                    as a second one would be half as many matrix instructions again:
//                    y is 2.1e-3 to 2.3e-3 from 64 bits, 1.7e-3 of it its own rounding)
// The running maximum is raised only when a score exceeds it by 2^8: the
// output is then rescaled (P stays below 256, its relative rounding does not
// change), which spares the rescaling of 64 accumulators on most tiles.
//
// Bound by the matrix and vector units, which take turns: matrix instructions
// are in work 48 % of the cycles, other vector ones 43 %, and the two waves of a
// SIMD hardly cover one's softmax with the other's products; neither operands
// read further ahead nor waves shifted against each other change the time.  LDS
// is active 25 % of the cycles by its counter; a wave of 32 rows reads an operand
// for every product, and 64 rows a wave, which would halve that, were not tried.
// The clock is 1.6 to 2.0 GHz under this load.  16 query
// heads on 4, d = 128: 16384 tokens without a window 1.05 to 1.09 PFLOP/s; 32768
// tokens, window 2048, 64 sinks 571 to 584 us, 950 TFLOP/s of visible products;
// B = 4, T = 4096, window 1024 (three of a row's 18 tiles are cut by the window
// or the diagonal, or hold the sinks) 152 us, 168 to 191 with y_low and lse.
template <int D>
__global__ void __launch_bounds__(256, 2) win_fwd_bf16_kernel(WinAttnArgs a) {
  using T = Tile<D>;
  constexpr int BK = 64, BYTES = BK * T::RB;
  // two buffers of K and V, each a variable of its own: what is read from one
  // then does not wait for the loads into the other
  __shared__ __attribute__((aligned(16))) char k0[BYTES], v0[BYTES], k1[BYTES], v1[BYTES];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, nt = (a.Tq * G + 127) / 128;
  // heads fastest (a head's tiles share an XCD's L2 where 8 divides the heads), the longest rows of keys first
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int part = w % a.parts, tile = nt - 1 - w / a.parts;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const RowMap rm(tile * 128, G, a.g_magic);
  const bf16* kb = (const bf16*)a.k + b * a.ks[0] + hk * a.ks[2];
  const bf16* vb = (const bf16*)a.v + b * a.vs[0] + hk * a.vs[2];

  // the wave's rows
  int qi, qh;
  rm.at(wave * 32 + n, &qi, &qh);
  qh += hk * G;
  const int p = qi < a.Tq && qi + off < len ? qi + off : -1;
  bf16x8 qf[T::NS];
  {
    const bf16* qp = (const bf16*)a.q + b * a.qs[0] + (long long)(p >= 0 ? qi : 0) * a.qs[1] + (long long)(p >= 0 ? qh : 0) * a.qs[2];
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      qf[c] = *(const bf16x8*)(qp + 16 * c + 8 * h);
      if (a.scale < 0.f) qf[c] = -qf[c];
    }
  }
  const float size = fabsf(a.scale) * kLog2e, sc = size < 1e-30f ? 1e-30f : size;      // (no number stays none)
  // positions of the workgroup's and of the wave's rows
  const int wg0 = rm.i0 + off, wg1 = min(rm.last(127), a.Tq - 1) + off;
  const int wv0 = rm.last(wave * 32) + off, wv1 = min(min(rm.last(wave * 32 + 31), a.Tq - 1) + off, len - 1);
  const bool rows_ok = rm.last(wave * 32 + 31) < a.Tq && rm.last(wave * 32 + 31) + off < len && wv0 >= 0;
  const KeyTiles<BK> kt(wg0, wg1, len, a.window, a.sinks);
  const int per = (kt.count + a.parts - 1) / a.parts, t0 = part * per, t1 = min(kt.count, t0 + per);

  f32x16 o[T::ND];
#pragma unroll
  for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  float m = -INFINITY, l = 0.f;

  const LaneMap<D> lm(lane);
  const TileLoad<D> tl(tid, wave, (int)a.ks[1], (int)a.vs[1]);
  const auto load = [&](char* tk, char* tv, int it) {
    const int j0 = kt.start(min(it, t1 - 1));
    tl.load(tk, kb + j0 * a.ks[1], tv, vb + j0 * a.vs[1], len - 1 - j0);
  };
  const auto tile_step = [&](const char* tk, const char* tv, int it) {
    const int j0 = kt.start(it);
    // whether the wave sees anything of the tile, and all of it
    const bool some = it < t1 && wv0 <= wv1 && j0 <= wv1 && (j0 + BK - 1 > wv0 - a.window || j0 < a.sinks);
    if (!some) return;
    const bool all = rows_ok && j0 + BK - 1 <= wv0 && (wv1 - j0 < a.window || j0 + BK <= a.sinks);
    f32x16 s[2];
    s[0] = s[1] = zero16();
    {                                      // (operands read two ahead: left alone, right before their use)
      bf16x8 fk[T::NS][2];
      const auto fetch = [&](int c) {
        fk[c][0] = lm.row(tk, c);
        fk[c][1] = lm.row(tk + 32 * T::RB, c);
      };
      fetch(0);
      fetch(1);
#pragma unroll
      for (int c = 0; c < T::NS; ++c) {
        __builtin_amdgcn_sched_barrier(0);
        if (c + 2 < T::NS) fetch(c + 2);
        mma32(s[0], fk[c][0], qf[c]);
        mma32(s[1], fk[c][1], qf[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!all) {
      const int d = p - j0 - 4 * h, ds = a.sinks - j0 - 4 * h;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = 32 * u + 8 * (e >> 2) + (e & 3);
          s[u][e] = (c <= d) & ((d - c < a.window) | (c < ds)) ? s[u][e] : -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
    mx = half_max(mx) * sc;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= f;
#pragma unroll
      for (int t = 0; t < T::ND; ++t) o[t] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], sc, -ms));
        sum += s[u][e];
      }
    l += sum;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 pf = acc_frag32(s[u], c);
#pragma unroll
        for (int t = 0; t < T::ND; ++t) mma32(o[t], lm.cols(tv + (32 * u + 16 * c) * T::RB, t), pf);
      }
  };
  if (t0 < t1) load(k0, v0, t0);
  loads_done_barrier();
  for (int it = t0; it < t1; it += 2) {
    load(k1, v1, it + 1);
    tile_step(k0, v0, it);
    loads_done_barrier();
    load(k0, v0, it + 2);
    tile_step(k1, v1, it + 1);
    loads_done_barrier();
  }
  l = half_sum(l);
  if (p < 0) {                             // a row that sees nothing: 0 times a value that is not finite is NaN
#pragma unroll
    for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  }
  // rows of the wave whose output is not finite (0 times it is NaN)
  float rest = 0.f;
#pragma unroll
  for (int t = 0; t < T::ND; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) rest = fmaf(o[t][e], 0.f, rest);
  const unsigned long long bad = __ballot(rest != 0.f);
  const unsigned redo = (unsigned)(bad | bad >> 32);
  if (a.parts > 1) {                       // a span of the keys: unnormalised, joined by win_join_kernel
    if (qi < a.Tq) {
      const long long r = ((long long)b * a.Tq + qi) * a.Hq + qh;
      float* po = part_out(a, part, r) + 4 * h;
#pragma unroll
      for (int t = 0; t < T::ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(po + 32 * t + 8 * i) = (f32x4){o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
      if (h == 0) {
        float* ml = part_stats(a, part, r);
        ml[0] = m;
        ml[1] = l;
      }
    }
    if (redo) {
      __builtin_amdgcn_s_waitcnt(0x0070);           // (the wave's own stores come first)
      careful_rows<bf16, D, BK, 32>(redo);
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (h == 0 && a.lse && qi < a.Tq)
    a.lse[((long long)b * a.Hq + qh) * a.Tq + qi] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
  // the output by way of LDS, so that whole rows are stored
  bf16* outs[2] = {(bf16*)a.y, (bf16*)a.y_low};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (!outs[m]) break;
    if (m) __syncthreads();
    lm.put((wave < 2 ? k0 : v0) + (wave & 1) * 32 * T::RB, o, inv, m == 1);
    __syncthreads();
    bf16* yb = outs[m] + (long long)b * a.Tq * a.Hq * D;
#pragma unroll
    for (int u = tid; u < 128 * T::UPR; u += 256) {
      const int r = u / T::UPR, c = u % T::UPR;
      int i, g;
      rm.at(r, &i, &g);
      if (i < a.Tq)
        *(uint4*)(yb + ((long long)i * a.Hq + hk * G + g) * D + 8 * c) = *(const uint4*)((r < 64 ? k0 : v0) + T::at(r & 63, c));
    }
  }
  if (__syncthreads_or(redo != 0) && redo) careful_rows<bf16, D, BK, 32>(redo);
}

template <int D> static int launch(const WinAttnArgs& a, hipStream_t stream) {
  const long long nt = ((long long)a.Tq * (a.Hq / a.Hkv) + 127) / 128;
  hipLaunchKernelGGL((win_fwd_bf16_kernel<D>), dim3((unsigned)(nt * a.B * a.Hkv * a.parts)), dim3(256), 0, stream, a);
  const int rc = check_launch("win_fwd_bf16_kernel");
  return rc ? rc : launch_win_join<bf16, D>(a, stream);
}

int win_fwd_bf16_dispatch(const WinAttnArgs& a, hipStream_t stream) {
  return a.D == 128 ? launch<128>(a, stream) : launch<64>(a, stream);
}

}  // namespace gdnx
