// Windowed attention with sinks for bf16 (gfx950): backward.  Forms and rules
// as in attn_win.hip, tiles and operands as in attn_tiles.hpp, rows packed as
// in the forward (attn_win_mfma.hip).
#include "attn_spans.hpp"
#include "attn_tiles.hpp"

namespace gdnx {

// dQ, and delta for dK: the forward's walk over the key tiles, per 32 x 32
// scores
//   S^T = K Q^T,  dP^T = V dY^T,  dS^T = P^T o (dP^T - delta),  dQ^T += K^T dS^T
// The scores are formed here and again by the dk / dv kernel, seven products in
// place of five: one kernel for all three would add its dq tiles up with float
// atomics, whose order changes the result, or write every tile's out.  P and dS
// are rounded to bf16 as the operands of the second products, as P is in the
// forward (gradients are 2.3e-3 to 2.4e-3 from 64 bits, 1.7e-3 of it their own
// rounding).  Bound like the forward (matrix instructions in work 43 % of the
// cycles, other vector ones 31 %, LDS 23 %); B = 4, T = 4096, 16/4 heads, d = 128,
// window 1024, 16 sinks: 225 to 254 us (448 thousand cycles; 480 with operands
// not read ahead).
template <int D>
__global__ void __launch_bounds__(256, 2) win_dq_bf16_kernel(WinAttnBwdArgs a) {
  using T = Tile<D>;
  constexpr int BK = 64, BYTES = BK * T::RB;
  __shared__ __attribute__((aligned(16))) char k0[BYTES], v0[BYTES], k1[BYTES], v1[BYTES];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, nt = (a.Tq * G + 127) / 128;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const int part = w % a.dq_parts, tile = nt - 1 - w / a.dq_parts;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk, off = a.Tk - a.Tq;
  const RowMap rm(tile * 128, G, a.g_magic);
  const bf16* kb = (const bf16*)a.k + b * a.ks[0] + hk * a.ks[2];
  const bf16* vb = (const bf16*)a.v + b * a.vs[0] + hk * a.vs[2];

  int qi, qh;
  rm.at(wave * 32 + n, &qi, &qh);
  qh += hk * G;
  const int p = qi < a.Tq && qi + off < len ? qi + off : -1;
  bf16x8 qf[T::NS], gf[T::NS];
  float delta = 0.f, lse = 0.f;
  {
    const int i = p >= 0 ? qi : 0, g = p >= 0 ? qh : 0;
    const bf16* qp = (const bf16*)a.q + b * a.qs[0] + (long long)i * a.qs[1] + (long long)g * a.qs[2];
    const long long row = (((long long)b * a.Tq + i) * a.Hq + g) * D;
    const long long srow = ((long long)b * a.Hq + g) * a.Tq + i;
#pragma unroll
    for (int c = 0; c < T::NS; ++c) {
      qf[c] = *(const bf16x8*)(qp + 16 * c + 8 * h);
      gf[c] = *(const bf16x8*)((const bf16*)a.dy + row + 16 * c + 8 * h);
      const bf16x8 yf = *(const bf16x8*)((const bf16*)a.y + row + 16 * c + 8 * h);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)gf[c][e] * (float)yf[e];
    }
    // (with y rounded to bf16 alone, delta's error would be that of dS over again)
    if (a.y_low)
#pragma unroll
      for (int c = 0; c < T::NS; ++c) {
        const bf16x8 yf = *(const bf16x8*)((const bf16*)a.y_low + row + 16 * c + 8 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)gf[c][e] * (float)yf[e];
      }
    delta = half_sum(delta);
    if (p >= 0) {
      lse = a.lse[srow] * kLog2e;
      if (h == 0 && part == 0) a.delta[srow] = delta;
    }
  }
  const float sc = a.scale * kLog2e;
  const int wg0 = rm.i0 + off, wg1 = min(rm.last(127), a.Tq - 1) + off;
  const int wv0 = rm.last(wave * 32) + off, wv1 = min(min(rm.last(wave * 32 + 31), a.Tq - 1) + off, len - 1);
  const bool rows_ok = rm.last(wave * 32 + 31) < a.Tq && rm.last(wave * 32 + 31) + off < len && wv0 >= 0;
  const KeyTiles<BK> kt(wg0, wg1, len, a.window, a.sinks);
  const int per = (kt.count + a.dq_parts - 1) / a.dq_parts, t0 = part * per, t1 = min(kt.count, t0 + per);

  f32x16 o[T::ND];
#pragma unroll
  for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  const LaneMap<D> lm(lane);
  const TileLoad<D> tl(tid, wave, (int)a.ks[1], (int)a.vs[1]);
  const auto load = [&](char* tk, char* tv, int it) {
    const int j0 = kt.start(min(it, t1 - 1));
    tl.load(tk, kb + j0 * a.ks[1], tv, vb + j0 * a.vs[1], len - 1 - j0);
  };
  const auto tile_step = [&](const char* tk, const char* tv, int it) {
    const int j0 = kt.start(it);
    const bool some = it < t1 && wv0 <= wv1 && j0 <= wv1 && (j0 + BK - 1 > wv0 - a.window || j0 < a.sinks);
    if (!some) return;
    const bool all = rows_ok && j0 + BK - 1 <= wv0 && (wv1 - j0 < a.window || j0 + BK <= a.sinks);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s = zero16(), dp = zero16();
      {                                    // (operands read one ahead: left alone, right before their use)
        bf16x8 fk[T::NS], fv[T::NS];
        const auto fetch = [&](int c) {
          fk[c] = lm.row(tk + u * 32 * T::RB, c);
          fv[c] = lm.row(tv + u * 32 * T::RB, c);
        };
        fetch(0);
#pragma unroll
        for (int c = 0; c < T::NS; ++c) {
          __builtin_amdgcn_sched_barrier(0);
          if (c + 1 < T::NS) fetch(c + 1);
          mma32(s, fk[c], qf[c]);
          mma32(dp, fv[c], gf[c]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], sc, -lse)) * (dp[e] - delta);
      if (!all) {
        const int d = p - j0 - 4 * h, ds = a.sinks - j0 - 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = 32 * u + 8 * (e >> 2) + (e & 3);
          s[e] = (c <= d) & ((d - c < a.window) | (c < ds)) ? s[e] : 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8 f = acc_frag32(s, c);
#pragma unroll
        for (int t = 0; t < T::ND; ++t) mma32(o[t], lm.cols(tk + (32 * u + 16 * c) * T::RB, t), f);
      }
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
  if (p < 0) {                             // a row that sees nothing: 0 times a key that is not finite is NaN
#pragma unroll
    for (int t = 0; t < T::ND; ++t) o[t] = zero16();
  }
  if (a.dq_parts > 1) {                    // a span of the keys: float32 sums, joined by win_dq_join_kernel
    if (qi < a.Tq) {
      float* po = a.part + (((long long)part * a.B + b) * a.Tq + qi) * a.Hq * D + qh * D + 4 * h;
#pragma unroll
      for (int t = 0; t < T::ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(po + 32 * t + 8 * i) = (f32x4){o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    }
    return;
  }
  lm.put((wave < 2 ? k0 : v0) + (wave & 1) * 32 * T::RB, o, a.scale);
  __syncthreads();
  bf16* qo = (bf16*)a.dq + (long long)b * a.Tq * a.Hq * D;
#pragma unroll
  for (int u = tid; u < 128 * T::UPR; u += 256) {
    const int r = u / T::UPR, c = u % T::UPR;
    int i, g;
    rm.at(r, &i, &g);
    if (i < a.Tq)
      *(uint4*)(qo + ((long long)i * a.Hq + hk * G + g) * D + 8 * c) = *(const uint4*)((r < 64 ? k0 : v0) + T::at(r & 63, c));
  }
}

// dK, dV of 128 keys of one key head over a span of the rows that see them; a
// wave owns 32 keys.  Per 32 rows
//   S = Q K^T,  dP = dY V^T,  dV^T += dY^T P,  dK^T += Q^T dS
// K stays in registers (the wave's 32 keys, half of what it holds are the sums),
// V in LDS, which both together would not fit beside; 32 rows of Q and dY a
// step, straight into LDS, double-buffered.  Bound by the latency of LDS: each
// product reads an operand, its waves wait 47 % of their cycles, LDS is active
// 30 % of all by its counter, and with two waves a SIMD the matrix units are busy
// 39 %.  B = 4, T = 4096, 16/4 heads, d = 128, window 1024, 16 sinks: 302 to 360 us
// (625 thousand cycles; 700 with operands not read ahead).
template <int D>
__global__ void __launch_bounds__(256, 2) win_dkv_bf16_kernel(WinAttnBwdArgs a) {
  using T = Tile<D>;
  constexpr int BR = 32, BYTES = BR * T::RB, VB = 128 * T::RB;
  __shared__ __attribute__((aligned(16))) char q0[BYTES], g0[BYTES], q1[BYTES], g1[BYTES], vtile[VB];
  __shared__ __attribute__((aligned(16))) float s_lse[2][BR], s_del[2][BR];
  __shared__ __attribute__((aligned(16))) int s_pos[2][BR];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.Hq / a.Hkv, off = a.Tk - a.Tq;
  int w = blockIdx.x;
  const int hk = w % a.Hkv; w /= a.Hkv;
  const int b = w % a.B; w /= a.B;
  const SpanSlot sl(a, w);
  const int part = sl.part, k0 = sl.tile * 128;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  const KeySpan<128> ks(a, k0, len);
  if (part >= ks.parts) return;
  const int t0 = part * ks.per * (64 / BR), t1 = min((part + 1) * ks.per * (64 / BR), (ks.rows + BR - 1) / BR);

  const int kw = k0 + wave * 32, j = kw + n;
  bf16x8 kf[T::NS];
  {
    const bf16* kp = (const bf16*)a.k + b * a.ks[0] + hk * a.ks[2] + (long long)max(0, min(j, len - 1)) * a.ks[1];
    const bf16* vp = (const bf16*)a.v + b * a.vs[0] + hk * a.vs[2];
#pragma unroll
    for (int c = 0; c < T::NS; ++c) kf[c] = *(const bf16x8*)(kp + 16 * c + 8 * h);
#pragma unroll
    for (int u = tid; u < 128 * T::UPR; u += 256) {
      const int r = u / T::UPR, c = u % T::UPR;
      *(u32x4*)(vtile + T::at(r, c)) =
          *(const u32x4*)(vp + (long long)max(0, min(k0 + r, len - 1)) * a.vs[1] + 8 * c);
    }
  }
  const float sc = a.scale * kLog2e;
  f32x16 ok[T::ND], ov[T::ND];
#pragma unroll
  for (int t = 0; t < T::ND; ++t) ok[t] = ov[t] = zero16();
  const bf16* qb = (const bf16*)a.q + b * a.qs[0] + (long long)hk * G * a.qs[2];
  const bf16* gb = (const bf16*)a.dy + ((long long)b * a.Tq * a.Hq + hk * G) * D;
  const LaneMap<D> lm_(lane);

  // step t: rows BR t .. of the keys' rows, clamped to the last one.  Q and dY
  // go straight into LDS, an instruction's 1 KB in lane order.
  constexpr int N = BR * T::UPR / 256, STEP = 256 / T::UPR;
  const int srow = tid / T::UPR, sunit = 8 * ((tid % T::UPR) ^ T::swz(srow));
  float x_lse = 0.f, x_del = 0.f;
  int x_pos = -1;
  const auto load = [&](char* tq, char* tg, const RowMap& rm, int t) {
    const int last = ks.rows - 1 - t * BR;
    typedef __attribute__((address_space(1))) void* Gp;
    typedef __attribute__((address_space(3))) void* Lp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int qi, qg;
      rm.at(min(srow + i * STEP, last), &qi, &qg);
      qi += ks.i0;
      __builtin_amdgcn_global_load_lds((Gp)(qb + qi * a.qs[1] + qg * a.qs[2] + sunit), (Lp)(tq + i * 4096 + wave * 1024),
                                       16, 0, 0);
      __builtin_amdgcn_global_load_lds((Gp)(gb + ((long long)qi * a.Hq + qg) * D + sunit),
                                       (Lp)(tg + i * 4096 + wave * 1024), 16, 0, 0);
    }
    if (tid < BR) {
      int qi, qg;
      rm.at(min(tid, last), &qi, &qg);
      qi += ks.i0;
      const long long sr = ((long long)b * a.Hq + hk * G + qg) * a.Tq + qi;
      x_lse = a.lse[sr];
      x_del = a.delta[sr];
      x_pos = tid <= last ? qi + off : -1;
    }
  };
  const auto store_stats = [&](int s) {
    if (tid < BR) {
      s_lse[s][tid] = x_lse * kLog2e;
      s_del[s][tid] = x_del;
      s_pos[s][tid] = x_pos;
    }
  };
  const char* vt = vtile + wave * 32 * T::RB;
  // tq, tg: the step's tiles, rm its rows; asks for the next step's into nq, ng
  RowMap rm(t0 * BR, G, a.g_magic);
  const auto row_step = [&](const char* tq, const char* tg, char* nq, char* ng, int t, int s_i) {
    const LaneMap<D> lm = lm_.fresh();
    // positions of the step's rows (uniform)
    const int tp0 = rm.i0 + ks.i0 + off, tp1 = rm.last(BR - 1) + ks.i0 + off;
    if (t + 1 < t1) {
      rm.advance(BR);
      load(nq, ng, rm, t + 1);
    }
    const bool some = tp1 >= kw && (tp0 - a.window < kw + 31 || kw < a.sinks);
    if (some) {
      const bool all = (t + 1) * BR <= ks.rows && tp0 >= kw + 31 && (tp1 - kw < a.window || kw + 32 <= a.sinks);
      f32x16 s = zero16(), dp = zero16();
      {
        bf16x8 fq[T::NS], fg[T::NS], fv[T::NS];
        const auto fetch = [&](int c) {
          fq[c] = lm.row(tq, c);
          fg[c] = lm.row(tg, c);
          fv[c] = lm.row(vt, c);
        };
        fetch(0);
#pragma unroll
        for (int c = 0; c < T::NS; ++c) {
          __builtin_amdgcn_sched_barrier(0);
          if (c + 1 < T::NS) fetch(c + 1);
          mma32(s, fq[c], kf[c]);
          mma32(dp, fg[c], fv[c]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 ls = *(const f32x4*)&s_lse[s_i][8 * q + 4 * h], dl = *(const f32x4*)&s_del[s_i][8 * q + 4 * h];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pr = __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], sc, -ls[e]));
          s[4 * q + e] = pr;
          dp[4 * q + e] = pr * (dp[4 * q + e] - dl[e]);
        }
      }
      if (!all) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int* ps = &s_pos[s_i][8 * q + 4 * h];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int p = ps[e];
            const bool vis = (j <= p) & ((p - j < a.window) | (j < a.sinks));
            s[4 * q + e] = vis ? s[4 * q + e] : 0.f;
            dp[4 * q + e] = vis ? dp[4 * q + e] : 0.f;
          }
        }
      }
      {
        constexpr int M = 2 * T::ND;
        bf16x8 fg[M], fq[M];
        const auto fetch = [&](int i) {
          fg[i] = lm.cols(tg + 16 * (i / T::ND) * T::RB, i % T::ND);
          fq[i] = lm.cols(tq + 16 * (i / T::ND) * T::RB, i % T::ND);
        };
        const bf16x8 pf[2] = {acc_frag32(s, 0), acc_frag32(s, 1)}, df[2] = {acc_frag32(dp, 0), acc_frag32(dp, 1)};
        fetch(0);
#pragma unroll
        for (int i = 0; i < M; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          if (i + 1 < M) fetch(i + 1);
          mma32(ov[i % T::ND], fg[i], pf[i / T::ND]);
          mma32(ok[i % T::ND], fq[i], df[i / T::ND]);
        }
      }
    }
    if (t + 1 < t1) store_stats(s_i ^ 1);
    loads_done_barrier();
  };
  if (t0 < t1) {
    load(q0, g0, rm, t0);
    store_stats(0);
  }
  loads_done_barrier();
  for (int t = t0; t < t1; t += 2) {
    row_step(q0, g0, q1, g1, t, 0);
    if (t + 1 < t1) row_step(q1, g1, q0, g0, t + 1, 1);
  }

  if (!key_seen(j, off, len, a.window, a.sinks)) {    // (0 times a query or dY that is not finite is NaN)
#pragma unroll
    for (int t = 0; t < T::ND; ++t) ok[t] = ov[t] = zero16();
  }
  if (ks.parts > 1) {                       // a span: float32 sums, joined by win_dkv_join_kernel
    const long long slot = ((long long)b * a.Hkv + hk) * span_slots<128>(a) + w;
    float* pk = a.part + (slot * 2 * 128 + wave * 32 + n) * D + 4 * h;
#pragma unroll
    for (int t = 0; t < T::ND; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *(f32x4*)(pk + 32 * t + 8 * i) = (f32x4){ok[t][4 * i], ok[t][4 * i + 1], ok[t][4 * i + 2], ok[t][4 * i + 3]};
        *(f32x4*)(pk + 128 * D + 32 * t + 8 * i) = (f32x4){ov[t][4 * i], ov[t][4 * i + 1], ov[t][4 * i + 2], ov[t][4 * i + 3]};
      }
    return;
  }
  // by way of LDS, so that whole rows are stored
  bf16* outs[2] = {(bf16*)a.dk, (bf16*)a.dv};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    __syncthreads();
    lm_.put(vtile + wave * 32 * T::RB, m ? ov : ok, m ? 1.f : a.scale);
    __syncthreads();
#pragma unroll
    for (int u = tid; u < 128 * T::UPR; u += 256) {
      const int r = u / T::UPR, c = u % T::UPR;
      if (k0 + r < a.Tk)
        *(uint4*)(outs[m] + (((long long)b * a.Tk + k0 + r) * a.Hkv + hk) * D + 8 * c) = *(const uint4*)(vtile + T::at(r, c));
    }
  }
}

template <int D> static int launch(const WinAttnBwdArgs& a, hipStream_t stream) {
  const long long heads = (long long)a.B * a.Hkv, nt = ((long long)a.Tq * (a.Hq / a.Hkv) + 127) / 128;
  hipLaunchKernelGGL((win_dq_bf16_kernel<D>), dim3((unsigned)(nt * heads * a.dq_parts)), dim3(256), 0, stream, a);
  int rc = check_launch("win_dq_bf16_kernel");
  if (rc || (rc = launch_dq_join<bf16>(a, stream))) return rc;
  hipLaunchKernelGGL((win_dkv_bf16_kernel<D>), dim3((unsigned)(span_slots<128>(a) * heads)), dim3(256), 0, stream, a);
  rc = check_launch("win_dkv_bf16_kernel");
  return rc ? rc : launch_dkv_join<bf16, D, 128>(a, stream);
}

int win_bwd_bf16_dispatch(const WinAttnBwdArgs& a, hipStream_t stream) {
  return a.D == 128 ? launch<128>(a, stream) : launch<64>(a, stream);
}

}  // namespace gdnx
