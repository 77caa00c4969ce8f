// Causal attention over texts laid end to end, forward, with shared key heads and an optional window with sinks:
//   O_i = sum_j P_ij V_j,  P_i = softmax over visible j of Q_i . K_j / sqrt(d),
//   visible: j <= p and (p - j < W or j < S), p = i + m - n the position of query i of n among its text's m keys;
// q, o [H, N, d], k, v [Hkv, M, d], query head h reads key head h / (H / Hkv).  Also writes the natural-log row sums
// (float32 [H, N], infinity for a query that sees no key) for the backward.
//
// Work is 4 d flops per visible pair: bound by the matrix cores.  A workgroup of four waves owns 128 queries of one text,
// 32 per wave with Q^T in registers, and walks the key tiles that one of them sees (window_attn.hip has the arrangement of
// a tile's products: S^T = K Q^T, so that the softmax is local to a lane and P^T the next product's operand as it stands).
// Tiles never cross texts: the keys behind a text's end are read as zeros.
// Where queries are few against the GPU, the key tiles are cut into chunks, a workgroup each, which leave unnormalised
// outputs with their maxima and sums to a second kernel.
// Measured, without the profiler's share: one text of 8192, 32(8)x128, 571 us (963 TFLOP/s); 12 texts to 4096, 32(8)x128, 700
// us (770: the ends of texts and of the grid); 3 texts to 10000, 16(2)x64, window 4000, 282 us (817: at 64 elements a head
// the exponentials take as long as the products); 8 texts of up to 64 queries on 28563 keys, 32(8)x128, 44 us, of which the
// chunks' kernel is 37 (3.2 TB/s of keys and values) and their join 6.5.
//
// Scores, softmax and O are float32.  In bf16 P is rounded to bf16 for the product (2^-8 of each term), and O's sum is that
// of the rounded values, so the weights of a row add to one.  For the backward, the row sums of partly hidden tiles, the
// only ones of a row of few keys, are those of P as it was (the others' roundings even out).  float32 runs on the float32
// matrix instructions.
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "edf_packed.hpp"

namespace edf {
namespace {

constexpr float LN2 = 0.6931471805599453f;

// Two workgroups a CU, three up to 64 elements a head where registers allow it; between 96 and 128 elements in bf16 5 registers
// are spilled, 14 where rows are read by elements.
template <typename T, int HD, int BN, bool VEC>
__global__ __launch_bounds__(256, (HD <= 64 ? 3 : 2)) void packed_fwd_kernel(PackArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32, NH = BN / 32;
  constexpr int AHEAD = sizeof(T) == 2 ? 4 : 1;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, l = tid & 63, g = l >> 5, li = l & 31;
  const QueryTile<BN> qt(a, sK);
  if (qt.none) return;
  const int d = a.d, myq = qt.myq, myp = qt.pw + li;
  const long row = qt.row0 + min(myq, qt.nq - 1);
  const T *K = (const T*)a.k + qt.krow * d, *V = (const T*)a.v + qt.krow * d;

  WFrag<T> qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) qf[kk] = window_row<T, HD, VEC>((const T*)a.q + row * d, kk * 16 + 8 * g, d);
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();
  float m = -INFINITY, lsum = 0.0f, lex = 0.0f;

  const TileLoader<T, HD, BN, VEC> ld(tid, d, qt.nk);
  WFrag<T> rk[ld.N], rv[ld.N];
  const int count = qt.t1 - qt.t0;
  auto gload = [&](int t) {
    ld.load(K, qt.key0(t), rk);
    ld.load(V, qt.key0(t), rv);
  };
  auto sstore = [&](int buf) {
    ld.template store<Tile>(sK[buf], rk);
    ld.template store<Tile>(sV[buf], rv);
  };
  auto tile = [&](int t, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const SeesKey sees(myp, qt.key0(t) + 4 * g, a.W, a.sinks);
    const T *sk = sK[t & 1], *sv = sV[t & 1];
    f32x16 s[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) s[h] = zero16();
    // consecutive products go to different halves' scores
    edf::ahead<NH * NKK, AHEAD>([&](int i) { return Tile::row(sk, i % NH * 32 + li, i / NH * 16 + 8 * g); },
                           [&](int i, const WFrag<T>& f) { s[i % NH] = WFrag<T>::mma(f, qf[i / NH], s[i % NH]); });
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (MASK) s[h][r] = sees(h * 32 + d_row(r, 0)) ? s[h][r] : -INFINITY;
        mx = fmaxf(mx, s[h][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    // O and the sum refer to a maximum that is moved only when a score exceeds it by a factor of 2^8: p <= 256 loses
    // nothing in float32 or bf16
    if (__any(mx * a.scale_log2 > m * a.scale_log2 + 8.0f)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = fast_exp2(m * a.scale_log2 - (mnew == -INFINITY ? 0.0f : mnew * a.scale_log2));
      lsum *= alpha;
      lex *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m = mnew;
    }
    const float mns = m == -INFINITY ? 0.0f : m * a.scale_log2;
    float rs = 0.0f, re = 0.0f;
    WFrag<T> pf[2 * NH];
#pragma unroll
    for (int kc = 0; kc < 2 * NH; ++kc)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int r = 8 * (kc & 1) + e;
        const float p0 = fast_exp2(fmaf(s[kc >> 1][r], a.scale_log2, -mns));
        const float p1 = fast_exp2(fmaf(s[kc >> 1][r + 1], a.scale_log2, -mns));
        rs = pf[kc].set2(e, p0, p1, rs);
        if constexpr (MASK && sizeof(T) == 2) re += p0 + p1;
      }
    rs += __shfl_xor(rs, 32);
    lsum += rs;
    lex += MASK && sizeof(T) == 2 ? re + __shfl_xor(re, 32) : rs;
    edf::ahead<2 * NH * NDT, AHEAD>([&](int i) { return Tile::trans(sv, 16 * (i / NDT), i % NDT, l); },
                               [&](int i, const WFrag<T>& f) { o[i % NDT] = WFrag<T>::mma(f, pf[i / NDT], o[i % NDT]); });
  };
  auto advance = [&](int t) {  // the next tile into the other buffer, the one after it into registers
    if (t + 1 < count) {
      sstore((t + 1) & 1);
      if (t + 2 < count) gload(t + 2);
    }
    __syncthreads();
  };
  if (count > 0) {
    gload(0);
    sstore(0);
    if (count > 1) gload(1);
  }
  __syncthreads();
  const int masked = min(count, max(qt.kt.first_whole - qt.t0, 0));
  int t = 0;
  for (; t < masked; ++t) {
    if (qt.visible(a, qt.key0(t), BN)) tile(t, std::true_type{});
    advance(t);
  }
  for (; t < count; ++t) {
    tile(t, std::false_type{});
    advance(t);
  }

  if (myq >= qt.nq) return;
  if (qt.slot >= 0) {
    float* out = a.part + qt.slot * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) =
            f32x4{o[dt][rb * 4], o[dt][rb * 4 + 1], o[dt][rb * 4 + 2], o[dt][rb * 4 + 3]};
    if (g == 0) {
      a.ml[3 * qt.slot] = m == -INFINITY ? -INFINITY : m * a.scale_log2;
      a.ml[3 * qt.slot + 1] = lsum;
      a.ml[3 * qt.slot + 2] = lex;
    }
    return;
  }
  const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;  // a query that sees no key answers with zeros
  T* O = (T*)a.out + row * d;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int c = dt * 32 + 8 * rb + 4 * g;
      if (VEC && c + 4 <= d) {
        typedef __attribute__((ext_vector_type(4))) T vec4;
        vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(o[dt][rb * 4 + e] * inv);
        *(vec4*)(O + c) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < d) O[c + e] = from_f32<T>(o[dt][rb * 4 + e] * inv);
      }
    }
  if (g == 0 && a.lse != nullptr)
    a.lse[row] = lex == 0.0f ? INFINITY : (m * a.scale_log2 + __log2f(lex)) * LN2;
}

// bf16 at head_dim 128: the same decomposition with tiles moved by 16-byte DMA loads into half-row-block LDS
// tiles (stage_hb: no staging registers, fragment addresses are bases plus immediates), two workgroups per CU,
// and K one tile ahead of V: the matrix products of the next tile's scores run between the exponentials of the
// current one wherever both are whole.
__global__ __launch_bounds__(256, 2) void packed_fwd128_kernel(PackArgs a) {
  constexpr int HD = 128, BN = 64, NKK = HD / 16, NDT = HD / 32;
  // X0 = {K buffer 0, V buffer 1}, X1 = {K buffer 1, V buffer 0}: iteration t (parity B) writes only X_B
  __shared__ __attribute__((aligned(16))) bf16 sX0[2 * BN * HD];
  __shared__ __attribute__((aligned(16))) bf16 sX1[2 * BN * HD];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  const QueryTile<BN> qt(a, sX0);
  if (qt.none) return;
  const int myp = qt.pw + li, myq = qt.myq;
  const bf16* Qrow = (const bf16*)a.q + (qt.row0 + min(myq, qt.nq - 1)) * HD;
  // buffer resources over the text's keys: rows past its end read as zeros (their scores are masked)
  const rsrc_t rK = make_rsrc((const bf16*)a.k + qt.krow * HD, (unsigned)qt.nk * HD * 2);
  const rsrc_t rV = make_rsrc((const bf16*)a.v + qt.krow * HD, (unsigned)qt.nk * HD * 2);

  bf16x8 qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) qf[kk] = *(const bf16x8*)(Qrow + kk * 16 + 8 * g);
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();
  float m = -INFINITY, lsum = 0.0f, lex = 0.0f;

  const int grp = l >> 4, i16 = l & 15;
  const int d0 = 16 * (grp & 1) + 4 * (i16 & 3), kr = 4 * (grp >> 1) + (i16 >> 2);
  const int krow[2] = {hb_row_base(li, g, 0), hb_row_base(li, g, 1)};
  const int vtr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  const int nkt = qt.t1 - qt.t0, whole = in_vector_register(max(qt.kt.first_whole - qt.t0, 0));
  auto visible = [&](int t) __attribute__((always_inline)) { return qt.visible(a, qt.key0(t), BN); };
  auto issue_k = [&](auto bt, int t) __attribute__((always_inline)) {
    stage_hb<BN>(rK, decltype(bt)::value ? sX1 : sX0, qt.key0(t), wu, l);
  };
  auto issue_v = [&](auto bt, int t) __attribute__((always_inline)) {
    stage_hb<BN>(rV, (decltype(bt)::value ? sX0 : sX1) + BN * HD, qt.key0(t), wu, l);
  };
  auto scores = [&](auto bt, f32x16* s) __attribute__((always_inline)) {
    const bf16* sk = decltype(bt)::value ? sX1 : sX0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = zero16();
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk)
        s[h] = mfma32(*(const bf16x8*)(&sk[krow[kk & 1] + hb_row_off<BN>(kk, 32 * h)]), qf[kk], s[h]);
    }
  };
  f32x16 sc[2], sn[2];  // scores of the current and the next tile
  // first half of the softmax: mask, row maximum, rescale; the maximum in scaled log2 units
  auto softmax_max = [&](f32x16* s, int t, auto masked) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(masked)::value;
    const SeesKey sees(myp, qt.key0(t) + 4 * g, a.W, a.sinks);
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (MASK) s[h][r] = sees(h * 32 + d_row(r, 0)) ? s[h][r] : -INFINITY;
        mx = fmaxf(mx, s[h][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    // O and the sum refer to a maximum that is moved only when a score exceeds it by a factor of 2^8: p <= 256
    // loses nothing in float32 or bf16
    if (__any(mx * a.scale_log2 > m * a.scale_log2 + 8.0f)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = fast_exp2(m * a.scale_log2 - (mnew == -INFINITY ? 0.0f : mnew * a.scale_log2));
      lsum *= alpha;
      lex *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m = mnew;
    }
    return m == -INFINITY ? 0.0f : m * a.scale_log2;
  };
  // second half for elements 2 j, 2 j + 1: p into the row sum and the P^T fragments.  pin: an empty volatile asm
  // keeps this arithmetic in the scheduling step that issued it.
  auto softmax_pair = [&](f32x16* s, int j, float mns, float& rs, float& re, bf16x8* pf, auto pin) __attribute__((always_inline)) {
    const int h = j >> 3, r = (2 * j) & 15;
    const float p0 = fast_exp2(fmaf(s[h][r], a.scale_log2, -mns)), p1 = fast_exp2(fmaf(s[h][r + 1], a.scale_log2, -mns));
    unsigned pk = pack_bf16x2(p0, p1);
    // the row sum of the bf16 P that the product consumes, one dot2 per pair
    rs = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk), bf16x2{(bf16)1.0f, (bf16)1.0f}, rs, false);
    if constexpr (decltype(pin)::value) asm volatile("" : "+v"(pk), "+v"(rs));
    else re += p0 + p1;
    const int kc = 2 * h + (r >> 3), it = r & 7;
    const bf16x2 pp = __builtin_bit_cast(bf16x2, pk);
    pf[kc][it] = pp[0];
    pf[kc][it + 1] = pp[1];
  };
  // O^T += V^T P^T: consecutive products go to different accumulators, V^T is read three steps ahead
  auto pv_mma = [&](auto bt, const bf16x8* pf) __attribute__((always_inline)) {
    const bf16* sv = (decltype(bt)::value ? sX0 : sX1) + BN * HD;
    auto vfrag = [&](int j) __attribute__((always_inline)) {
      const int o16 = hb_tr_off<BN>(j & 3, j >> 2, 0);
      return cat4(lds_read_tr16(&sv[vtr[0] + o16]), lds_read_tr16(&sv[vtr[1] + o16]));
    };
    bf16x8 v[3] = {vfrag(0), vfrag(1), vfrag(2)};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      o[j & 3] = mfma32(v[j % 3], pf[j >> 2], o[j & 3]);
      if (j + 3 < 16) v[j % 3] = vfrag(j + 3);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto consume = [&](auto bt, f32x16* s, int t, auto masked) __attribute__((always_inline)) {
    const float mns = softmax_max(s, t, masked);
    float rs = 0.0f, re = 0.0f;
    bf16x8 pf[4];
#pragma unroll
    for (int j = 0; j < 16; ++j) softmax_pair(s, j, mns, rs, re, pf, std::false_type{});
    lsum += rs + __shfl_xor(rs, 32);
    lex += re + __shfl_xor(re, 32);
    pv_mma(bt, pf);
  };
  // whole tile t with a successor: the 16 products of S(t + 1) alternate with the exponentials of S(t)
  auto fused = [&](auto bt, int t) __attribute__((always_inline)) {
    const bf16* sk = decltype(bt)::value ? sX0 : sX1;
    const float mns = softmax_max(sc, t, std::false_type{});
    auto kfrag = [&](int i) __attribute__((always_inline)) {
      const int kk = i >> 1;
      return *(const bf16x8*)(&sk[krow[kk & 1] + hb_row_off<BN>(kk, 32 * (i & 1))]);
    };
    bf16x8 fr[4] = {kfrag(0), kfrag(1), kfrag(2), kfrag(3)};
    sn[0] = zero16();
    sn[1] = zero16();
    float rs = 0.0f;
    bf16x8 pf[4];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sn[i & 1] = mfma32(fr[i & 3], qf[i >> 1], sn[i & 1]);
      if (i + 4 < 16) fr[i & 3] = kfrag(i + 4);
      softmax_pair(sc, i, mns, rs, rs, pf, std::true_type{});
      __builtin_amdgcn_sched_barrier(0);
    }
    rs += __shfl_xor(rs, 32);
    lsum += rs;
    lex += rs;
    pv_mma(bt, pf);
  };
  const std::integral_constant<int, 0> b0{};
  const std::integral_constant<int, 1> b1{};
  if (nkt > 0) {
    issue_k(b0, 0);
    issue_v(b0, 0);
  }
  wait_vm();
  if (nkt > 1) issue_k(b1, 1);
  __syncthreads();  // K(0), V(0) visible
  if (nkt > 0 && visible(0)) scores(b0, sc);
  wait_vm();
  __syncthreads();  // K(1) visible, K buffer 0 free
  // iteration t (buffer parity B = t % 2): K(t + 2) into K buffer B, V(t + 1) into V buffer 1 - B
  auto step = [&](auto bt, int t) __attribute__((always_inline)) {
    const std::integral_constant<int, 1 - decltype(bt)::value> ot{};
    if (t + 2 < nkt) issue_k(bt, t + 2);
    if (t + 1 < nkt) issue_v(ot, t + 1);
    const bool next = t + 1 < nkt;
    if (t >= whole && next) {
      fused(bt, t);
    } else {
      if (next && visible(t + 1)) scores(ot, sn);
      if (t >= whole) consume(bt, sc, t, std::false_type{});
      else if (visible(t)) consume(bt, sc, t, std::true_type{});
    }
    wait_vm();
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) sc[h] = sn[h];
  };
  for (int t = 0; t < nkt; t += 2) {
    step(b0, t);
    if (t + 1 < nkt) step(b1, t + 1);
  }

  if (qt.slot >= 0) {
    if (myq >= qt.nq) return;
    float* out = a.part + qt.slot * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) =
            f32x4{o[dt][rb * 4], o[dt][rb * 4 + 1], o[dt][rb * 4 + 2], o[dt][rb * 4 + 3]};
    if (g == 0) {
      a.ml[3 * qt.slot] = m == -INFINITY ? -INFINITY : m * a.scale_log2;
      a.ml[3 * qt.slot + 1] = lsum;
      a.ml[3 * qt.slot + 2] = lex;
    }
    return;
  }
  // O through the free array X0 (each wave its 32 rows), written as whole rows
  bf16* so = sX0 + w * 32 * HD;
  const float inv = myq >= qt.nq || lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      bf16x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (bf16)(o[dt][rb * 4 + e] * inv);
      *(bf16x4*)(so + lds_off<HD>(li, dt * 32 + 8 * rb + 4 * g)) = v;
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = l + 64 * i, row = e / 16, ch = e % 16;
    if (myq - li + row < qt.nq)
      *(bf16x8*)((bf16*)a.out + (qt.row0 + myq - li + row) * HD + 8 * ch) = *(const bf16x8*)(so + lds_off<HD>(row, 8 * ch));
  }
  if (myq < qt.nq && g == 0 && a.lse != nullptr)
    a.lse[qt.row0 + myq] = lex == 0.0f ? INFINITY : (m * a.scale_log2 + __log2f(lex)) * LN2;
}

// The chunks of a row joined: out = sum_c 2^(m_c - m) O_c / sum_c 2^(m_c - m) l_c, four elements a lane.
template <typename T, int HD>
__global__ __launch_bounds__(256) void packed_join_kernel(PackArgs a) {
  constexpr int LANES = HD <= 32 ? 8 : HD <= 64 ? 16 : 32;
  const ChunkRow<LANES> r(a);
  if (r.chunks == 0) return;
  const int j = threadIdx.x % LANES, e = 4 * j;
  const float* ml = a.ml + 3 * r.slot;
  float m = -INFINITY, sum = 0.0f, exact = 0.0f;
  for (int c = j; c < r.chunks; c += LANES) m = fmaxf(m, ml[3L * PK_M * c]);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* in = a.part + r.slot * HD + min(e, HD - 4);
#pragma unroll 4
  for (int c = 0; c < r.chunks; ++c) {
    const float mc = ml[3L * PK_M * c], f = mc == -INFINITY ? 0.0f : fast_exp2(mc - m);
    sum = fmaf(f, ml[3L * PK_M * c + 1], sum);
    exact = fmaf(f, ml[3L * PK_M * c + 2], exact);
    acc += f * *(const f32x4*)(in + (long)PK_M * HD * c);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < a.d) st((T*)a.out, r.row * a.d + e + i, acc[i] * inv);
  if (j == 0 && a.lse != nullptr) a.lse[r.row] = exact == 0.0f ? INFINITY : (m + __log2f(exact)) * LN2;
}

template <typename T, int HD, int BN, bool VEC>
int launch_fwd(hipStream_t s, PackArgs a) {
  const long groups = a.H >> a.hs, grid = packed_grid(groups, a.items > 0 ? a.items : a.nx);
  bool done = false;
  if constexpr (sizeof(T) == 2 && HD == 128 && VEC) {
    if (a.d == 128) {
      packed_fwd128_kernel<<<(unsigned)grid, 256, 0, s>>>(a);
      done = true;
    }
  }
  if (!done) packed_fwd_kernel<T, HD, BN, VEC><<<(unsigned)grid, 256, 0, s>>>(a);
  if (a.items > 0)
    packed_join_kernel<T, HD><<<(unsigned)packed_grid(groups, (long)a.nx * (HD <= 32 ? 4 : HD <= 64 ? 8 : 16)), 256, 0, s>>>(a);
  return check_launch("packed attention");
}
template <typename T, int BN, bool VEC>
int launch_fwd_d(hipStream_t s, const PackArgs& a) {
  switch (window_pad(a.d)) {
    case 32: return launch_fwd<T, 32, BN, VEC>(s, a);
    case 64: return launch_fwd<T, 64, BN, VEC>(s, a);
    case 96: return launch_fwd<T, 96, BN, VEC>(s, a);
    default: return launch_fwd<T, 128, BN, VEC>(s, a);
  }
}

}  // namespace

int packed_check(int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim, int window, int sinks,
                 int dtype) {
  EDF_REQUIRE(num_heads > 0 && num_kv_heads > 0 && rows > 0 && key_rows > 0 && head_dim > 0 && texts >= 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(num_heads % num_kv_heads == 0, EDF_ERR_INVALID_ARG, "num_heads %d is no multiple of num_kv_heads %d",
              num_heads, num_kv_heads);
  EDF_REQUIRE(window >= 0 && sinks >= 0, EDF_ERR_INVALID_ARG, "window and sinks must not be negative");
  EDF_REQUIRE(head_dim <= 128, EDF_ERR_UNSUPPORTED, "head_dim %d > 128 unsupported", head_dim);
  // a key, a window of 2^30 and a tile past it together stay an int
  EDF_REQUIRE(rows < (1L << 29) && key_rows < (1L << 29) && texts < (1 << 28) && sinks < (1 << 29), EDF_ERR_UNSUPPORTED,
              "rows, keys and sinks must be below 2^29, texts below 2^28");
  EDF_REQUIRE((double)num_heads * packed_tiles(std::max(rows, key_rows), texts, 32) * 4 < 2147483648.0, EDF_ERR_UNSUPPORTED,
              "heads x rows too large for one call");
  return EDF_OK;
}

}  // namespace edf

extern "C" {

size_t edf_packed_attention_workspace_bytes(int num_heads, int num_kv_heads, long rows, long key_rows, int texts,
                                            int head_dim, int window, int sinks, int dtype) {
  using namespace edf;
  if (packed_check(num_heads, num_kv_heads, rows, key_rows, texts, head_dim, window, sinks, dtype)) return 0;
  PackArgs a{};
  a.N = (int)rows, a.M = (int)key_rows, a.S = texts, a.H = num_heads, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window > 0 ? std::min(window, PK_ALL) : PK_ALL, a.sinks = sinks;
  query_plan(a, key_tile(dtype));
  return chunk_bytes(a, 3);
}

int edf_packed_attention(void* stream, const void* q, const void* k, const void* v, const int32_t* offsets,
                         const int32_t* key_offsets, void* out, float* lse, void* workspace, size_t workspace_bytes,
                         int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim, int window,
                         int sinks, int dtype) {
  using namespace edf;
  const int rc = packed_check(num_heads, num_kv_heads, rows, key_rows, texts, head_dim, window, sinks, dtype);
  if (rc) return rc;
  EDF_REQUIRE(q && k && v && offsets && key_offsets && out, EDF_ERR_INVALID_ARG, "null tensor pointer");
  PackArgs a{};
  a.q = q, a.k = k, a.v = v, a.qo = offsets, a.ko = key_offsets, a.out = out, a.lse = lse;
  a.N = (int)rows, a.M = (int)key_rows, a.S = texts, a.H = num_heads, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window > 0 ? std::min(window, PK_ALL) : PK_ALL, a.sinks = sinks;
  a.scale = 1.0f / sqrtf((float)head_dim), a.scale_log2 = a.scale * LOG2E;
  query_plan(a, key_tile(dtype));
  const size_t need = chunk_bytes(a, 3);
  EDF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), EDF_ERR_WORKSPACE,
              "workspace too small: need %zu bytes", need);
  chunk_memory(a, (float*)workspace, 3);
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out;
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15) && key_rows <= WINDOW_VEC_T;
  hipStream_t s = as_stream(stream);
  if (dtype == EDF_BF16) return vec ? launch_fwd_d<bf16, 64, true>(s, a) : launch_fwd_d<bf16, 64, false>(s, a);
  return vec ? launch_fwd_d<float, 32, true>(s, a) : launch_fwd_d<float, 32, false>(s, a);
}

}  // extern "C"
