// Attention with a sliding window and sinks, backward (window_attn.hip has the forward and its formulas):
//   P from the forward's row sums; dV_j = sum_i P_ij dO_i, dP = dO V^T, D_i = dO_i . O_i,
//   dS = P (dP - D) / sqrt(d), dQ = dS K, dK = dS^T Q; dK, dV summed over the query heads of a key head.
// 10 d flops per visible pair (S and dP formed twice, once for each kernel): bound by the matrix cores.
//
//   dQ: a workgroup owns 128 queries (32 per wave, Q^T and dO^T in registers) and walks the key tiles of
//   the forward; it also forms D and leaves it for the second kernel.
//   dK, dV: a workgroup owns 128 keys (32 per wave, K^T and V^T in registers) of one key head and walks the
//   query tiles that see one of them, query head by query head: the sum over shared heads needs no atomics.
//   Keys that hold sinks are seen by every later query, T / 64 tiles a head instead of (W + 128) / 64, and
//   with few keys and heads there are fewer workgroups than the GPU holds: such a block's tiles are then
//   divided over several workgroups, each leaving float32 sums, added in order by a third kernel.  Where that
//   is less, the queries past the windows meet the sinks in a kernel of their own (window_narrow.hip).
// In bf16 P and dS are rounded as operands of the second products (2^-8 of each term), D is formed from the rounded O
// that the forward left, and P from the forward's sum of rounded probabilities: a row's P is off as a whole by the mean
// of their roundings, at most 2^-8 of itself, where one probability far above the others is not at the maximum that the
// sums refer to.  Everything else is float32.  On random inputs (300 rows, window 100) the 2-norm of dQ is 1.65e-3 off by
// its own rounding, as much by that of dS, 0.8e-3 by D and 0.3e-3 by the row sums: 2.5e-3 together.  dS in two bf16
// parts would be two of the seven products again, D from an unrounded O a float32 O to keep until the backward, a second
// sum of the unrounded P 32 additions a tile in the forward, whose vector instructions bound it.
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "edf_window.hpp"

namespace edf {
int window_check(int batch, int num_heads, int num_kv_heads, int seq_len, int head_dim, int window, int sinks,
                 int dtype);
namespace {

constexpr int WB_M = 128;  // queries (dQ) or keys (dK, dV) per workgroup

template <typename T, int HD, int BN, bool VEC>
__global__ __launch_bounds__(256, 1) void window_dq_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32, NH = BN / 32;
  constexpr int AHEAD = sizeof(T) == 2 ? 3 : 1;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (a.nx - 1 - xb) * WB_M, qw = q0 + 32 * w, myq = qw + li;
  const long qrow = bh * T_ + min(myq, T_ - 1);
  const T* K = (const T*)a.k + bh / a.G * T_ * d;
  const T* V = (const T*)a.v + bh / a.G * T_ * d;

  WFrag<T> qf[NKK], of[NKK];
  float dd = 0.0f;
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const int col = kk * 16 + 8 * g;
    qf[kk] = window_row<T, HD, VEC>((const T*)a.q + qrow * d, col, d);
    of[kk] = window_row<T, HD, VEC>((const T*)a.go + qrow * d, col, d);
    const WFrag<T> oo = window_row<T, HD, VEC>((const T*)a.o + qrow * d, col, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) dd = fmaf(oo.get(e), of[kk].get(e), dd);
  }
  dd += __shfl_xor(dd, 32);
  const float lse = a.lse[qrow] * LOG2E;
  if (g == 0 && myq < T_) a.dd[qrow] = dd;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zero16();

  const KeyTiles<WB_M, BN> kt(q0, T_, a.W, a.S);
  const TileLoader<T, HD, BN, VEC> ld(tid, d, T_);
  WFrag<T> rk[ld.N], rv[ld.N];
  auto gload = [&](int t) {
    const int k0 = kt.key0(t);
    ld.load(K, k0, rk);
    ld.load(V, k0, rv);
  };
  auto sstore = [&](int buf) {
    ld.template store<Tile>(sK[buf], rk);
    ld.template store<Tile>(sV[buf], rv);
  };
  auto tile = [&](int t, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const SeesKey sees(myq, kt.key0(t) + 4 * g, a.W, a.S);
    const T *sk = sK[t & 1], *sv = sV[t & 1];
    f32x16 s[NH], dp[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      s[h] = zero16();
      dp[h] = zero16();
    }
    ahead<NH * NKK, AHEAD>(
        [&](int i) {
          const int row = i / NKK * 32 + li, col = i % NKK * 16 + 8 * g;
          return Pair<T>{Tile::row(sk, row, col), Tile::row(sv, row, col)};
        },
        [&](int i, const Pair<T>& f) {
          s[i / NKK] = WFrag<T>::mma(f.x, qf[i % NKK], s[i / NKK]);
          dp[i / NKK] = WFrag<T>::mma(f.y, of[i % NKK], dp[i / NKK]);
        });
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = fast_exp2(fmaf(s[h][r], a.scale_log2, -lse)) * (dp[h][r] - dd);  // 1 / sqrt(d) at the end
        if constexpr (MASK) x = sees(h * 32 + d_row(r, 0)) ? x : 0.0f;
        s[h][r] = x;
      }
    WFrag<T> df[2 * NH];
#pragma unroll
    for (int kc = 0; kc < 2 * NH; ++kc)
#pragma unroll
      for (int e = 0; e < 8; ++e) df[kc].set(e, s[kc >> 1][8 * (kc & 1) + e]);
    ahead<2 * NH * NDT, AHEAD>([&](int i) { return Tile::trans(sk, 16 * (i / NDT), i % NDT, l); },
                               [&](int i, const WFrag<T>& f) { dq[i % NDT] = WFrag<T>::mma(f, df[i / NDT], dq[i % NDT]); });
  };
  auto advance = [&](int t) {
    if (t + 1 < kt.count) {
      sstore((t + 1) & 1);
      if (t + 2 < kt.count) gload(t + 2);
    }
    __syncthreads();
  };
  gload(0);
  sstore(0);
  if (kt.count > 1) gload(1);
  __syncthreads();
  int t = 0;
  for (; t < kt.first_whole; ++t) {
    const int k0 = kt.key0(t);
    if ((k0 <= qw + 31 && k0 + BN + a.W > qw + 1) || k0 < a.S) tile(t, std::true_type{});
    advance(t);
  }
  for (; t < kt.count; ++t) {
    tile(t, std::false_type{});
    advance(t);
  }
  if (myq >= T_) return;
  T* out = (T*)a.dq + qrow * d;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int c = dt * 32 + 8 * rb + 4 * g;
      if (VEC && c + 4 <= d) {
        typedef __attribute__((ext_vector_type(4))) T vec4;
        vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(dq[dt][rb * 4 + e] * a.scale);
        *(vec4*)(out + c) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < d) out[c + e] = from_f32<T>(dq[dt][rb * 4 + e] * a.scale);
      }
    }
}

// dQ, bf16 at head_dim 128: tiles by DMA loads, each as two 32-key halves so that one half's S and dP are live;
// two workgroups per CU, so one wave's exponentials and waits overlap another's products.
__global__ __launch_bounds__(256, 2) void window_dq128_kernel(WindowArgs a) {
  constexpr int HD = 128, BN = 64, NKK = HD / 16, NDT = HD / 32;
  __shared__ __attribute__((aligned(16))) bf16 sR0[2 * BN * HD];  // ring slot: K then V
  __shared__ __attribute__((aligned(16))) bf16 sR1[2 * BN * HD];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T = a.T;
  const int q0 = (a.nx - 1 - xb) * WB_M, qw = q0 + 32 * w, myq = qw + li;
  const long qrow = bh * T + min(myq, T - 1), kvbase = bh / a.G * T * HD;
  const rsrc_t rK = make_rsrc((const bf16*)a.k + kvbase, (unsigned)T * HD * 2);
  const rsrc_t rV = make_rsrc((const bf16*)a.v + kvbase, (unsigned)T * HD * 2);

  bf16x8 qf[NKK], of[NKK];
  float dd = 0.0f;
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const long at = qrow * HD + kk * 16 + 8 * g;
    qf[kk] = *(const bf16x8*)((const bf16*)a.q + at);
    of[kk] = *(const bf16x8*)((const bf16*)a.go + at);
    const bf16x8 ov = *(const bf16x8*)((const bf16*)a.o + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) dd = fmaf((float)of[kk][e], (float)ov[e], dd);
  }
  dd += __shfl_xor(dd, 32);
  const float lse = a.lse[qrow] * LOG2E;
  if (g == 0 && myq < T) a.dd[qrow] = dd;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zero16();

  const int grp = l >> 4, i16 = l & 15;
  const int d0 = 16 * (grp & 1) + 4 * (i16 & 3), kr = 4 * (grp >> 1) + (i16 >> 2);
  const int krow[2] = {hb_row_base(li, g, 0), hb_row_base(li, g, 1)};
  const int ktr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  const KeyTiles<WB_M, BN> kt(q0, T, a.W, a.S);
  const int whole = in_vector_register(kt.first_whole);
  auto issue = [&](auto bt, int t) {
    constexpr int B = decltype(bt)::value;
    const int k0 = kt.key0(t);
    stage_hb<BN>(rK, B ? sR1 : sR0, k0, wu, l);
    stage_hb<BN>(rV, (B ? sR1 : sR0) + BN * HD, k0, wu, l);
  };
  auto tile = [&](auto bt, int t, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const bf16* sK = decltype(bt)::value ? sR1 : sR0;
    const bf16* sV = sK + BN * HD;
    const int k0 = kt.key0(t);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kb = k0 + 32 * h;
      if (MASK && !((kb <= qw + 31 && kb + 32 + a.W > qw + 1) || kb < a.S)) continue;  // no visible pair
      const SeesKey sees(myq, kb + 4 * g, a.W, a.S);
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        const int off = krow[kk & 1] + hb_row_off<BN>(kk, 32 * h);
        s = mfma32(*(const bf16x8*)(&sK[off]), qf[kk], s);
        dp = mfma32(*(const bf16x8*)(&sV[off]), of[kk], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = fast_exp2(fmaf(s[r], a.scale_log2, -lse)) * (dp[r] - dd);
        if constexpr (MASK) x = sees(d_row(r, 0)) ? x : 0.0f;
        s[r] = x;
      }
      bf16x8 df[2];
#pragma unroll
      for (int kc = 0; kc < 2; ++kc)
#pragma unroll
        for (int e = 0; e < 8; ++e) df[kc][e] = (bf16)s[8 * kc + e];
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          const int o = hb_tr_off<BN>(dt, kc, 32 * h);
          dq[dt] = mfma32(cat4(lds_read_tr16(&sK[ktr[0] + o]), lds_read_tr16(&sK[ktr[1] + o])), df[kc], dq[dt]);
        }
    }
  };
  auto step = [&](auto bt, int t) {
    const std::integral_constant<int, 1 - decltype(bt)::value> ot{};
    if (t + 1 < kt.count) issue(ot, t + 1);
    if (t >= whole) tile(bt, t, std::false_type{});
    else tile(bt, t, std::true_type{});
    wait_vm();
    __syncthreads();
  };
  const std::integral_constant<int, 0> b0{};
  const std::integral_constant<int, 1> b1{};
  issue(b0, 0);
  wait_vm();
  __syncthreads();
  for (int t = 0; t < kt.count; t += 2) {
    step(b0, t);
    if (t + 1 < kt.count) step(b1, t + 1);
  }
  if (myq >= T) return;
  bf16* out = (bf16*)a.dq + qrow * HD;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (bf16)(dq[dt][rb * 4 + e] * a.scale);
      *(bf16x4*)(out + dt * 32 + 8 * rb + 4 * g) = v;
    }
}

// bf16 widths to 96 keep to 256 registers, two workgroups a CU (at 96 with 24 of them spilled, and one load step less
// ahead: 4x16(4)x1500x80 window 400 backward 157 -> 144 us).
template <typename T, int HD, int BQ, bool VEC>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && HD <= 96 && VEC ? 2 : 1)) void window_dkdv_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  constexpr int AHEAD = sizeof(T) == 4 ? 1 : HD == 96 ? 2 : 3;
  using Tile = WTile<T, HD, BQ>;
  __shared__ __attribute__((aligned(16))) T sQ[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sO[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) float sL[2][BQ], sD[2][BQ];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;  // batch x key head
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const KeyChunk<WB_M, BQ> kc_(a, xb, bh);
  const int kb0 = kc_.key0, kw = kb0 + 32 * w, mykey = kw + li, qs = kc_.qs, nt = kc_.nt, t0 = kc_.t0, t1 = kc_.t1;

  const T* K = (const T*)a.k + bh * T_ * d;
  const T* V = (const T*)a.v + bh * T_ * d;
  WFrag<T> kf[NKK], vf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const long row = (long)min(mykey, T_ - 1) * d;
    kf[kk] = window_row<T, HD, VEC>(K + row, kk * 16 + 8 * g, d);
    vf[kk] = window_row<T, HD, VEC>(V + row, kk * 16 + 8 * g, d);
  }
  f32x16 dk[NDT], dv[NDT];  // dK^T, dV^T: rows are dims, the column this lane's key
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    dk[dt] = zero16();
    dv[dt] = zero16();
  }
  const TileLoader<T, HD, BQ, VEC> ld(tid, d, T_);
  WFrag<T> rq[ld.N], ro[ld.N];
  float rl = 0.0f, rd = 0.0f;
  auto gload = [&](int t) {
    const int h = t / nt, q0 = qs + (t - h * nt) * BQ;
    const long base = (bh * a.G + h) * T_;
    ld.load((const T*)a.q + base * d, q0, rq);
    ld.load((const T*)a.go + base * d, q0, ro);
    if (tid < BQ) {
      const long q = base + min(q0 + tid, T_ - 1);
      rl = q0 + tid < T_ ? a.lse[q] * LOG2E : INFINITY;  // a query past the end gets P = 0
      rd = a.dd[q];
    }
  };
  auto sstore = [&](int buf) {
    ld.template store<Tile>(sQ[buf], rq);
    ld.template store<Tile>(sO[buf], ro);
    if (tid < BQ) {
      sL[buf][tid] = rl;
      sD[buf][tid] = rd;
    }
  };
  if (t0 < t1) {
    gload(t0);
    sstore(0);
    if (t0 + 1 < t1) gload(t0 + 1);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const int q0 = qs + t % nt * BQ;
#pragma unroll
    for (int sub = 0; sub < BQ / 32; ++sub) {
      const int qb = q0 + 32 * sub;
      // no query of the sub-tile sees a key of this wave
      if (qb + 31 < kw || (qb > kw + 30 + a.W && kw >= a.S)) continue;
      auto subtile = [&](auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        f32x16 s = zero16(), dp = zero16();
        ahead<NKK, AHEAD>(
            [&](int i) {
              const int row = 32 * sub + li, col = i * 16 + 8 * g;
              return Pair<T>{Tile::row(sQ[buf], row, col), Tile::row(sO[buf], row, col)};
            },
            [&](int i, const Pair<T>& f) {
              s = WFrag<T>::mma(f.x, kf[i], s);
              dp = WFrag<T>::mma(f.y, vf[i], dp);
            });
#pragma unroll
        for (int rb = 0; rb < 4; ++rb) {
          const f32x4 lv = *(const f32x4*)(&sL[buf][32 * sub + 8 * rb + 4 * g]);
          const f32x4 dv4 = *(const f32x4*)(&sD[buf][32 * sub + 8 * rb + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = rb * 4 + e;
            float p = fast_exp2(fmaf(s[r], a.scale_log2, -lv[e]));
            float x = p * (dp[r] - dv4[e]);  // 1 / sqrt(d) is applied to dK at the end
            if constexpr (MASK) {
              const bool see = window_sees(qb + 8 * rb + 4 * g + e, mykey, a.W, a.S);
              p = see ? p : 0.0f;
              x = see ? x : 0.0f;
            }
            s[r] = p;
            dp[r] = x;
          }
        }
        WFrag<T> pf[2], df[2];
#pragma unroll
        for (int kc = 0; kc < 2; ++kc)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pf[kc].set(e, s[8 * kc + e]);
            df[kc].set(e, dp[8 * kc + e]);
          }
        ahead<2 * NDT, AHEAD>(
            [&](int i) {
              const int r0 = 32 * sub + 16 * (i / NDT);
              return Pair<T>{Tile::trans(sO[buf], r0, i % NDT, l), Tile::trans(sQ[buf], r0, i % NDT, l)};
            },
            [&](int i, const Pair<T>& f) {
              dv[i % NDT] = WFrag<T>::mma(f.x, pf[i / NDT], dv[i % NDT]);
              dk[i % NDT] = WFrag<T>::mma(f.y, df[i / NDT], dk[i % NDT]);
            });
      };
      // every pair visible: the queries lie past the wave's keys and within the window of its first
      if (qb >= kw + 31 && qb + 31 - kw < a.W) subtile(std::false_type{});
      else subtile(std::true_type{});
    }
    if (t + 1 < t1) {
      sstore(buf ^ 1);
      if (t + 2 < t1) gload(t + 2);
    }
    __syncthreads();
  }
  if (kc_.slot >= 0) {  // these sums are a part: [dK | dV][key][dim] of the block
    float* out = a.part + kc_.slot * (2L * WB_M * HD) + (32 * w + li) * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        f32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = dk[dt][rb * 4 + e];
          y[e] = dv[dt][rb * 4 + e];
        }
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) = x;
        *(f32x4*)(out + WB_M * HD + dt * 32 + 8 * rb + 4 * g) = y;
      }
    return;
  }
  if (mykey >= T_) return;
  T* krow = (T*)a.dk + (bh * T_ + mykey) * d;
  T* vrow = (T*)a.dv + (bh * T_ + mykey) * d;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int c = dt * 32 + 8 * rb + 4 * g;
      if (VEC && c + 4 <= d) {
        typedef __attribute__((ext_vector_type(4))) T vec4;
        vec4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = from_f32<T>(dk[dt][rb * 4 + e] * a.scale);
          y[e] = from_f32<T>(dv[dt][rb * 4 + e]);
        }
        *(vec4*)(krow + c) = x;
        *(vec4*)(vrow + c) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < d) {
            krow[c + e] = from_f32<T>(dk[dt][rb * 4 + e] * a.scale);
            vrow[c + e] = from_f32<T>(dv[dt][rb * 4 + e]);
          }
      }
    }
}

// dK, dV, bf16 at head_dim 128: V is read from an LDS copy of the workgroup's 128 keys (its fragments would not
// fit 256 registers beside the two accumulators), Q and dO come in 32-query tiles by DMA loads, two workgroups per
// CU.
__global__ __launch_bounds__(256, 2) void window_dkdv128_kernel(WindowArgs a) {
  constexpr int HD = 128, BQ = 32, NKK = HD / 16, NDT = HD / 32;
  __shared__ __attribute__((aligned(16))) bf16 sV[WB_M * HD];
  __shared__ __attribute__((aligned(16))) bf16 sR0[2 * BQ * HD];  // ring slot: Q then dO
  __shared__ __attribute__((aligned(16))) bf16 sR1[2 * BQ * HD];
  __shared__ __attribute__((aligned(16))) float sL0[BQ], sL1[BQ], sD0[BQ], sD1[BQ];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  int xb;
  long bh;  // batch x key head
  window_block(a, xb, bh);
  const int T = a.T;
  const KeyChunk<WB_M, BQ> kc_(a, xb, bh);
  const int kb0 = kc_.key0, kw = kb0 + 32 * w, mykey = kw + li, qs = kc_.qs, nt = kc_.nt, t0 = kc_.t0, t1 = kc_.t1;

  // keys past the end read zero rows of V: they only feed their own columns, never stored
  stage_hb<WB_M>(make_rsrc((const bf16*)a.v + bh * T * HD, (unsigned)T * HD * 2), sV, kb0, wu, l);
  bf16x8 kf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk)
    kf[kk] = *(const bf16x8*)((const bf16*)a.k + (bh * T + min(mykey, T - 1)) * HD + kk * 16 + 8 * g);
  f32x16 dk[NDT], dv[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    dk[dt] = zero16();
    dv[dt] = zero16();
  }
  float rl = 0.0f, rd = 0.0f;
  // Tile t into ring slot B: Q and dO by DMA, row sums and D into registers of the first wave, which publish()
  // writes to LDS once the tile's loads have landed.
  auto issue = [&](auto bt, int t) {
    constexpr int B = decltype(bt)::value;
    const int h = t / nt, q0 = qs + (t - h * nt) * BQ;
    const long row = (bh * a.G + h) * T;
    stage_hb<BQ>(make_rsrc((const bf16*)a.q + row * HD, (unsigned)T * HD * 2), B ? sR1 : sR0, q0, wu, l);
    stage_hb<BQ>(make_rsrc((const bf16*)a.go + row * HD, (unsigned)T * HD * 2), (B ? sR1 : sR0) + BQ * HD, q0, wu, l);
    if (tid < BQ) {
      const long q = row + min(q0 + tid, T - 1);
      rl = q0 + tid < T ? a.lse[q] : INFINITY;  // a query past the end gets P = 0
      rd = a.dd[q];
    }
  };
  auto publish = [&](auto bt) {
    constexpr int B = decltype(bt)::value;
    wait_vm();
    if (tid < BQ) {
      (B ? sL1 : sL0)[tid] = rl * LOG2E;
      (B ? sD1 : sD0)[tid] = rd;
    }
  };
  const int grp = l >> 4, i16 = l & 15;
  const int d0 = 16 * (grp & 1) + 4 * (i16 & 3), kr = 4 * (grp >> 1) + (i16 >> 2);
  const int qrow[2] = {hb_row_base(li, g, 0), hb_row_base(li, g, 1)};
  const int vrow[2] = {hb_row_base(li, g, 0) + hb_row_off<WB_M>(0, 32 * w),
                       hb_row_base(li, g, 1) + hb_row_off<WB_M>(0, 32 * w)};
  const int qtr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  auto subtile = [&](auto bt, int qb, auto masked) {
    constexpr int B = decltype(bt)::value;
    constexpr bool MASK = decltype(masked)::value;
    const bf16* sQ = B ? sR1 : sR0;
    const bf16* sO = sQ + BQ * HD;
    // distinct barriers keep the two bodies' equal LDS reads from being hoisted above their branch
    __builtin_amdgcn_sched_barrier(MASK ? 1 : 2);
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int off = qrow[kk & 1] + hb_row_off<BQ>(kk, 0);
      const bf16x8 vf = *(const bf16x8*)(&sV[vrow[kk & 1] + hb_row_off<WB_M>(kk, 0)]);
      s = mfma32(*(const bf16x8*)(&sQ[off]), kf[kk], s);
      dp = mfma32(*(const bf16x8*)(&sO[off]), vf, dp);
    }
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const f32x4 lv = *(const f32x4*)(&(B ? sL1 : sL0)[8 * rb + 4 * g]);
      const f32x4 dv4 = *(const f32x4*)(&(B ? sD1 : sD0)[8 * rb + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = rb * 4 + e;
        float p = fast_exp2(fmaf(s[r], a.scale_log2, -lv[e]));
        float x = p * (dp[r] - dv4[e]);
        if constexpr (MASK) {
          const bool see = window_sees(qb + 8 * rb + 4 * g + e, mykey, a.W, a.S);
          p = see ? p : 0.0f;
          x = see ? x : 0.0f;
        }
        s[r] = p;
        dp[r] = x;
      }
    }
    bf16x8 pf[2], df[2];
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pf[kc][e] = (bf16)s[8 * kc + e];
        df[kc][e] = (bf16)dp[8 * kc + e];
      }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const int o = hb_tr_off<BQ>(dt, kc, 0);
        dv[dt] = mfma32(cat4(lds_read_tr16(&sO[qtr[0] + o]), lds_read_tr16(&sO[qtr[1] + o])), pf[kc], dv[dt]);
        dk[dt] = mfma32(cat4(lds_read_tr16(&sQ[qtr[0] + o]), lds_read_tr16(&sQ[qtr[1] + o])), df[kc], dk[dt]);
      }
  };
  auto step = [&](auto bt, int t) {
    const std::integral_constant<int, 1 - decltype(bt)::value> ot{};
    if (t + 1 < t1) issue(ot, t + 1);
    const int qb = qs + t % nt * BQ;
    if (!(qb + 31 < kw || (qb > kw + 30 + a.W && kw >= a.S))) {  // some query sees a key of this wave
      if (qb >= kw + 31 && qb + 31 - kw < a.W) subtile(bt, qb, std::false_type{});
      else subtile(bt, qb, std::true_type{});
    }
    if (t + 1 < t1) publish(ot);
    __syncthreads();
  };
  const std::integral_constant<int, 0> b0{};
  const std::integral_constant<int, 1> b1{};
  if (t0 < t1) {
    issue(b0, t0);
    publish(b0);
  } else {
    wait_vm();
  }
  __syncthreads();
  for (int t = t0; t < t1; t += 2) {
    step(b0, t);
    if (t + 1 < t1) step(b1, t + 1);
  }
  if (kc_.slot >= 0) {  // these sums are a part: [dK | dV][key][dim] of the block
    float* out = a.part + kc_.slot * (2L * WB_M * HD) + (32 * w + li) * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        f32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = dk[dt][rb * 4 + e];
          y[e] = dv[dt][rb * 4 + e];
        }
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) = x;
        *(f32x4*)(out + WB_M * HD + dt * 32 + 8 * rb + 4 * g) = y;
      }
    return;
  }
  if (mykey >= T) return;
  const long row = (bh * T + mykey) * HD;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      bf16x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = (bf16)(dk[dt][rb * 4 + e] * a.scale);
        y[e] = (bf16)dv[dt][rb * 4 + e];
      }
      *(bf16x4*)((bf16*)a.dk + row + dt * 32 + 8 * rb + 4 * g) = x;
      *(bf16x4*)((bf16*)a.dv + row + dt * 32 + 8 * rb + 4 * g) = y;
    }
}

constexpr int BQ_BF16 = 64, BQ_32 = 32;  // query tiles: bf16, and float32 or the DMA kernel

template <typename T, int HD, int BN, int BQ, bool VEC>
int launch_bwd(hipStream_t s, WindowArgs a, int BH, int BHkv) {
  a.nx = (a.T + WB_M - 1) / WB_M;
  const unsigned grid = (unsigned)a.nx * (unsigned)BH;
  constexpr bool dma = sizeof(T) == 2 && HD == 128 && VEC;
  const bool fast = dma && a.d == 128;
  int rc = EDF_OK;
  if (window_narrow(BH, a.T, VEC)) {
    rc = window_narrow_run(true, s, a, BH, sizeof(T) == 2 ? EDF_BF16 : EDF_F32);
  } else {
    if (fast) window_dq128_kernel<<<grid, 256, 0, s>>>(a);
    else window_dq_kernel<T, HD, BN, VEC><<<grid, 256, 0, s>>>(a);
    rc = check_launch("window attention dQ");
  }
  if (rc) return rc;
  if constexpr (dma) {
    if (fast) return launch_dkdv<bf16, 128, WB_M, BQ_32, VEC>(s, a, BHkv, window_dkdv128_kernel);
  }
  return launch_dkdv<T, HD, WB_M, BQ, VEC>(s, a, BHkv, window_dkdv_kernel<T, HD, BQ, VEC>);
}


template <typename T, int BN, int BQ, bool VEC>
int launch_bwd_d(hipStream_t s, const WindowArgs& a, int BH, int BHkv) {
  switch (window_pad(a.d)) {
    case 32: return launch_bwd<T, 32, BN, BQ, VEC>(s, a, BH, BHkv);
    case 64: return launch_bwd<T, 64, BN, BQ, VEC>(s, a, BH, BHkv);
    case 96: return launch_bwd<T, 96, BN, BQ, VEC>(s, a, BH, BHkv);
    default: return launch_bwd<T, 128, BN, BQ, VEC>(s, a, BH, BHkv);
  }
}

}  // namespace
}  // namespace edf

extern "C" {

size_t edf_window_attention_backward_workspace_bytes(int batch, int num_heads, int num_kv_heads, int seq_len,
                                                     int head_dim, int window, int sinks, int dtype) {
  using namespace edf;
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || seq_len <= 0 || head_dim <= 0 || window <= 0 || sinks < 0)
    return 0;
  const int W = std::min(window, seq_len), S = std::min(sinks, seq_len), heads = batch * num_kv_heads;
  const size_t rows = ((size_t)batch * num_heads * seq_len * sizeof(float) + 255) & ~(size_t)255;
  // of the largest of the plans that may run: which one does also depends on the tensors' alignment
  size_t sums = 0;
  auto need = [&](int kb, int bq) {
    const int hd = window_pad(head_dim), G = num_heads / num_kv_heads;
    const KvPlan p = dtype == EDF_BF16
                         ? kv_plan(heads, G, seq_len, W, S, hd, kb, bq, 2, kv_slots<bf16>(hd), kv_join<bf16>(kb, bq))
                         : kv_plan(heads, G, seq_len, W, S, hd, kb, bq, 4, kv_slots<float>(hd), kv_join<float>(kb, bq));
    sums = std::max(sums, heads * (p.part(kb, hd) + p.far(hd)) * sizeof(float));
  };
  need(WB_M, BQ_32);
  if (dtype == EDF_BF16) need(WB_M, BQ_BF16);
  return rows + sums;
}

int edf_window_attention_backward(void* stream, const void* q, const void* k, const void* v, const void* out,
                                  const void* grad_out, const float* lse, void* grad_q, void* grad_k, void* grad_v,
                                  void* workspace, size_t workspace_bytes, int batch, int num_heads,
                                  int num_kv_heads, int seq_len, int head_dim, int window, int sinks, int dtype) {
  using namespace edf;
  const int rc = window_check(batch, num_heads, num_kv_heads, seq_len, head_dim, window, sinks, dtype);
  if (rc) return rc;
  EDF_REQUIRE(q && k && v && out && grad_out && lse && grad_q && grad_k && grad_v, EDF_ERR_INVALID_ARG,
              "null tensor pointer (the forward's lse is required)");
  const size_t need = edf_window_attention_backward_workspace_bytes(batch, num_heads, num_kv_heads, seq_len, head_dim,
                                                                    window, sinks, dtype);
  EDF_REQUIRE(workspace && workspace_bytes >= need, EDF_ERR_WORKSPACE, "workspace too small: need %zu bytes", need);
  WindowArgs a{};
  a.q = q, a.k = k, a.v = v, a.o = out, a.go = grad_out, a.lse = const_cast<float*>(lse);
  a.dq = grad_q, a.dk = grad_k, a.dv = grad_v, a.dd = (float*)workspace;
  const size_t rows = ((size_t)batch * num_heads * seq_len * sizeof(float) + 255) & ~(size_t)255;
  a.part = (float*)((char*)workspace + rows);
  a.T = seq_len, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window < seq_len ? window : seq_len, a.S = sinks < seq_len ? sinks : seq_len;
  a.scale = 1.0f / sqrtf((float)head_dim), a.scale_log2 = a.scale * LOG2E;
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)grad_out |
                         (uintptr_t)grad_q | (uintptr_t)grad_k | (uintptr_t)grad_v;
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15) && seq_len <= WINDOW_VEC_T;
  hipStream_t s = as_stream(stream);
  const int BH = batch * num_heads, BHkv = batch * num_kv_heads;
  if (dtype == EDF_BF16)
    return vec ? launch_bwd_d<bf16, 64, BQ_BF16, true>(s, a, BH, BHkv)
               : launch_bwd_d<bf16, 64, BQ_BF16, false>(s, a, BH, BHkv);
  return vec ? launch_bwd_d<float, 32, BQ_32, true>(s, a, BH, BHkv)
             : launch_bwd_d<float, 32, BQ_32, false>(s, a, BH, BHkv);
}

}  // extern "C"
