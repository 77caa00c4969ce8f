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
//   divided over several workgroups, each leaving float32 sums, added in order by a third kernel.
// P and dS are rounded to bf16 as operands of the second products (2^-8 of each term); everything else is
// float32.
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
  constexpr int CPR = HD / 8, PIECES = BN * CPR, CPT = (PIECES + 255) / 256;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  head_block(xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (gridDim.x - 1 - xb) * WB_M, qw = q0 + 32 * w, myq = qw + li;
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
  WFrag<T> rk[CPT], rv[CPT];
  auto gload = [&](int t) {
    const int k0 = kt.key0(t);
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      const long key = min(k0 + row, T_ - 1);  // rows past the end repeat the last: their P is masked
      rk[i] = window_row<T, HD, VEC>(K + key * d, col, d);
      rv[i] = window_row<T, HD, VEC>(V + key * d, col, d);
    }
  };
  auto sstore = [&](int buf) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      rk[i].store(&sK[buf][Tile::off(row, col)]);
      rv[i].store(&sV[buf][Tile::off(row, col)]);
    }
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
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        s[h] = WFrag<T>::mma(Tile::row(sk, h * 32 + li, kk * 16 + 8 * g), qf[kk], s[h]);
        dp[h] = WFrag<T>::mma(Tile::row(sv, h * 32 + li, kk * 16 + 8 * g), of[kk], dp[h]);
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = fast_exp2(fmaf(s[h][r], a.scale_log2, -lse)) * (dp[h][r] - dd);  // 1 / sqrt(d) at the end
        if constexpr (MASK) x = sees(h * 32 + d_row(r, 0)) ? x : 0.0f;
        s[h][r] = x;
      }
#pragma unroll
    for (int kc = 0; kc < 2 * NH; ++kc) {
      WFrag<T> df;
#pragma unroll
      for (int e = 0; e < 8; ++e) df.set(e, s[kc >> 1][8 * (kc & 1) + e]);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) dq[dt] = WFrag<T>::mma(Tile::trans(sk, 16 * kc, dt, l), df, dq[dt]);
    }
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
  head_block(xb, bh);
  const int T = a.T;
  const int q0 = (gridDim.x - 1 - xb) * WB_M, qw = q0 + 32 * w, myq = qw + li;
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

// Query tiles of BQ that see a key of block [k0, k0 + WB_M): from qs on, n of them per query head.
template <int BQ>
EDF_DEVICE void query_tiles(int k0, int T, int W, int S, int& qs, int& n) {
  qs = k0;
  const int end = k0 < S ? T : min(T, k0 + WB_M - 1 + W);  // one past the last query
  n = (end - qs + BQ - 1) / BQ;
}

template <typename T, int HD, int BQ, bool VEC>
__global__ __launch_bounds__(256, 1) void window_dkdv_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  constexpr int CPR = HD / 8, PIECES = BQ * CPR, CPT = (PIECES + 255) / 256;
  using Tile = WTile<T, HD, BQ>;
  __shared__ __attribute__((aligned(16))) T sQ[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sO[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) float sL[2][BQ], sD[2][BQ];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;  // batch x key head
  head_block(xb, bh);
  const int T_ = a.T, d = a.d;
  // which key block, and which of its chunks of tiles
  const bool sink_part = xb < a.nsb * a.c_sink;
  const int xr = sink_part ? xb : xb - a.nsb * a.c_sink;
  const int per = sink_part ? a.c_sink : a.c_win, len = sink_part ? a.len_sink : a.len_win;
  const int kblk = (sink_part ? 0 : a.nsb) + xr / per, chunk = xr % per;
  const int kb0 = kblk * WB_M, kw = kb0 + 32 * w, mykey = kw + li;
  int qs, nt;
  query_tiles<BQ>(kb0, T_, a.W, a.S, qs, nt);
  const int t0 = chunk * len, t1 = min(t0 + len, nt * a.G);  // tiles (query head, tile) of this workgroup

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
  WFrag<T> rq[CPT], ro[CPT];
  float rl = 0.0f, rd = 0.0f;
  auto gload = [&](int t) {
    const int h = t / nt, q0 = qs + (t - h * nt) * BQ;
    const long base = (bh * a.G + h) * T_;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      const long q = base + min(q0 + row, T_ - 1);  // rows past the end repeat the last: their P is 0
      rq[i] = window_row<T, HD, VEC>((const T*)a.q + q * d, col, d);
      ro[i] = window_row<T, HD, VEC>((const T*)a.go + q * d, col, d);
    }
    if (tid < BQ) {
      const long q = base + min(q0 + tid, T_ - 1);
      rl = q0 + tid < T_ ? a.lse[q] * LOG2E : INFINITY;
      rd = a.dd[q];
    }
  };
  auto sstore = [&](int buf) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      rq[i].store(&sQ[buf][Tile::off(row, col)]);
      ro[i].store(&sO[buf][Tile::off(row, col)]);
    }
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
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
          s = WFrag<T>::mma(Tile::row(sQ[buf], 32 * sub + li, kk * 16 + 8 * g), kf[kk], s);
          dp = WFrag<T>::mma(Tile::row(sO[buf], 32 * sub + li, kk * 16 + 8 * g), vf[kk], dp);
        }
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
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
          WFrag<T> pf, df;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pf.set(e, s[8 * kc + e]);
            df.set(e, dp[8 * kc + e]);
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            dv[dt] = WFrag<T>::mma(Tile::trans(sO[buf], 32 * sub + 16 * kc, dt, l), pf, dv[dt]);
            dk[dt] = WFrag<T>::mma(Tile::trans(sQ[buf], 32 * sub + 16 * kc, dt, l), df, dk[dt]);
          }
        }
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
  if (per > 1) {  // this chunk's sums: [dK | dV][key][dim] of the block
    float* out = a.part + (bh * (long)gridDim.x + xb) * (2L * WB_M * HD) + (32 * w + li) * HD;
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
  head_block(xb, bh);
  const int T = a.T;
  const bool sink_part = xb < a.nsb * a.c_sink;
  const int xr = sink_part ? xb : xb - a.nsb * a.c_sink;
  const int per = sink_part ? a.c_sink : a.c_win, len = sink_part ? a.len_sink : a.len_win;
  const int kblk = (sink_part ? 0 : a.nsb) + xr / per, chunk = xr % per;
  const int kb0 = kblk * WB_M, kw = kb0 + 32 * w, mykey = kw + li;
  int qs, nt;
  query_tiles<BQ>(kb0, T, a.W, a.S, qs, nt);
  const int t0 = chunk * len, t1 = min(t0 + len, nt * a.G);

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
  if (per > 1) {  // this chunk's sums: [dK | dV][key][dim] of the block
    float* out = a.part + (bh * (long)gridDim.x + xb) * (2L * WB_M * HD) + (32 * w + li) * HD;
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

// dK, dV of the blocks that were divided: the chunks' sums added in order, four elements a thread.  Grid x:
// pieces of the block's [dK | dV][key][dim], y: the divided blocks from `first` on, z: batch x key head.
template <typename T, int HD, int BQ>
__global__ __launch_bounds__(256) void window_sum_kernel(WindowArgs a, int gx, int first, int per) {
  const int kblk = first + blockIdx.y, kb0 = kblk * WB_M;
  const long bh = blockIdx.z;
  int qs, nt;
  query_tiles<BQ>(kb0, a.T, a.W, a.S, qs, nt);
  const int len = kblk < a.nsb ? a.len_sink : a.len_win;
  const int n = min(per, (nt * a.G + len - 1) / len);  // chunks that hold a tile
  const int x0 = kblk < a.nsb ? kblk * a.c_sink : a.nsb * a.c_sink + (kblk - a.nsb) * a.c_win;
  const int e = (blockIdx.x * 256 + threadIdx.x) * 4;
  const bool is_v = e >= WB_M * HD;
  const int key = e / HD % WB_M, c = e % HD;
  if (kb0 + key >= a.T || c >= a.d) return;
  const float* in = a.part + (bh * gx + x0) * (2L * WB_M * HD) + e;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int i = 0; i < n; ++i) s += *(const f32x4*)(in + i * (2L * WB_M * HD));
  if (!is_v) s *= a.scale;
  T* out = (T*)(is_v ? a.dv : a.dk) + (bh * a.T + kb0 + key) * a.d + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < a.d) out[i] = from_f32<T>(s[i]);
}

constexpr int WB_FILL = 512;  // workgroups of the dK, dV kernel that fill the GPU twice over

struct KvPlan {
  int nkb, nsb, c_sink, c_win, len_sink, len_win;
  int gx() const { return nsb * c_sink + (nkb - nsb) * c_win; }
};
// How many workgroups share a key block's tiles: one where the blocks alone fill the GPU, else as many as fill
// it; a sink block's tiles are divided into chunks no longer than another block's.
KvPlan kv_plan(int heads, int G, int T, int W, int S, int BQ) {
  KvPlan p;
  p.nkb = (T + WB_M - 1) / WB_M;
  p.nsb = std::min(p.nkb, (S + WB_M - 1) / WB_M);
  const long n_sink = (long)G * ((T + BQ - 1) / BQ);
  const long n_win = std::min(n_sink, (long)G * ((WB_M - 1 + W + BQ - 1) / BQ));
  const long want = std::max(1L, WB_FILL / std::max(1L, (long)p.nkb * heads));
  p.c_win = (int)std::min(want, n_win);
  p.len_win = (int)((n_win + p.c_win - 1) / p.c_win);
  p.c_win = (int)((n_win + p.len_win - 1) / p.len_win);
  // (many sink keys: no more workgroups, each with its float32 sums, than fill the GPU four times over)
  const long all = n_sink * p.nsb * heads;
  p.len_sink = (int)std::max((long)p.len_win, (all + 4 * WB_FILL - 1) / (4 * WB_FILL));
  p.c_sink = (int)std::max(1L, (n_sink + p.len_sink - 1) / p.len_sink);
  return p;
}

// the dK, dV kernel of the call, its query tiles, and the sums of divided blocks
template <typename T, int HD, int BQ, typename F>
int launch_dkdv(hipStream_t s, WindowArgs a, int BHkv, F kernel) {
  const KvPlan p = kv_plan(BHkv, a.G, a.T, a.W, a.S, BQ);
  a.nsb = p.nsb, a.c_sink = p.c_sink, a.c_win = p.c_win, a.len_sink = p.len_sink, a.len_win = p.len_win;
  const int gx = p.gx();
  kernel<<<dim3(gx, BHkv), 256, 0, s>>>(a);
  const int rc = check_launch("window attention dK, dV");
  if (rc) return rc;
  if (p.nsb > 0 && p.c_sink > 1)
    window_sum_kernel<T, HD, BQ><<<dim3(2 * WB_M * HD / 1024, p.nsb, BHkv), 256, 0, s>>>(a, gx, 0, p.c_sink);
  if (p.nkb > p.nsb && p.c_win > 1)
    window_sum_kernel<T, HD, BQ><<<dim3(2 * WB_M * HD / 1024, p.nkb - p.nsb, BHkv), 256, 0, s>>>(a, gx, p.nsb, p.c_win);
  return check_launch("window attention dK, dV sums");
}

constexpr int BQ_BF16 = 64, BQ_32 = 32;  // query tiles: bf16, and float32 or the DMA kernel
bool dma_kernels(int d, int T, int dtype, bool vec) { return dtype == EDF_BF16 && vec && d == 128 && T <= WINDOW_DMA_T; }

template <typename T, int HD, int BN, int BQ, bool VEC>
int launch_bwd(hipStream_t s, WindowArgs a, int BH, int BHkv) {
  const dim3 grid((a.T + WB_M - 1) / WB_M, BH);
  constexpr bool dma = sizeof(T) == 2 && HD == 128 && VEC;
  const bool fast = dma && dma_kernels(a.d, a.T, EDF_BF16, VEC);
  if (fast) window_dq128_kernel<<<grid, 256, 0, s>>>(a);
  else window_dq_kernel<T, HD, BN, VEC><<<grid, 256, 0, s>>>(a);
  const int rc = check_launch("window attention dQ");
  if (rc) return rc;
  if constexpr (dma) {
    if (fast) return launch_dkdv<bf16, 128, BQ_32>(s, a, BHkv, window_dkdv128_kernel);
  }
  return launch_dkdv<T, HD, BQ>(s, a, BHkv, window_dkdv_kernel<T, HD, BQ, VEC>);
}

int pad_width(int d) { return (d + 31) / 32 * 32; }

template <typename T, int BN, int BQ, bool VEC>
int launch_bwd_d(hipStream_t s, const WindowArgs& a, int BH, int BHkv) {
  switch (pad_width(a.d)) {
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
  size_t sums = 0;  // of the larger of the plans: which kernel runs also depends on the tensors' alignment
  for (int bq : {BQ_BF16, BQ_32}) {
    const KvPlan p = kv_plan(heads, num_heads / num_kv_heads, seq_len, W, S, bq);
    if ((dtype == EDF_BF16 || bq == BQ_32) && ((p.nsb > 0 && p.c_sink > 1) || (p.nkb > p.nsb && p.c_win > 1)))
      sums = std::max(sums, (size_t)heads * p.gx() * 2 * WB_M * pad_width(head_dim) * sizeof(float));
  }
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
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15);
  hipStream_t s = as_stream(stream);
  const int BH = batch * num_heads, BHkv = batch * num_kv_heads;
  if (dtype == EDF_BF16)
    return vec ? launch_bwd_d<bf16, 64, BQ_BF16, true>(s, a, BH, BHkv)
               : launch_bwd_d<bf16, 64, BQ_BF16, false>(s, a, BH, BHkv);
  return vec ? launch_bwd_d<float, 32, BQ_32, true>(s, a, BH, BHkv)
             : launch_bwd_d<float, 32, BQ_32, false>(s, a, BH, BHkv);
}

}  // extern "C"
