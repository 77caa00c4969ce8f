// Attention with a sliding window and sinks, forward, with shared key heads:
//   O_i = sum_j P_ij V_j,  P_i = softmax over visible j of Q_i . K_j / sqrt(d),
//   visible: j <= i and (i - j < W or j < S);  q, o [B, Hq, T, d], k, v [B, Hkv, T, d], query head h reads
// key head h / (Hq / Hkv).  Also writes the natural-log row sums (float32 [B, Hq, T]) for the backward.
//
// Work is 4 d flops per visible pair, about T W pairs a head: bound by the matrix cores.  A workgroup of
// four waves owns 128 queries, 32 per wave with Q^T in registers, and walks only the key tiles that one of
// them sees: S^T = K Q^T puts a query into a lane's column, so the softmax is local to the lane plus one
// exchange, and the registers of P^T are the operand of O^T += V^T P^T as they stand.  Tiles are
// double-buffered in LDS with the next one on its way in registers.  The partly hidden tiles come first
// (one loop with the mask), the others after it (one loop without): the order of an online softmax is free.
//
// Scores, softmax and O are float32.  In bf16 P is rounded to bf16 for the product (2^-8 of each term), and its sum is
// that of the rounded values, here and in the narrow kernels, so the weights of a row add to one; the row sums that the
// backward takes are the same (window_attn_bwd.hip has what that adds).  float32 runs on the float32 matrix instructions.
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "edf_window.hpp"

namespace edf {
namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr int WA_BM = 128;

template <typename T, int HD, int BN, bool VEC>
__global__ __launch_bounds__(256, 2) void window_fwd_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32, NH = BN / 32;
  constexpr int AHEAD = sizeof(T) == 2 ? 4 : 1;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (a.nx - 1 - xb) * WA_BM, qw = q0 + 32 * w, myq = qw + li;
  const T* Q = (const T*)a.q + bh * T_ * d;
  const T* K = (const T*)a.k + bh / a.G * T_ * d;
  const T* V = (const T*)a.v + bh / a.G * T_ * d;

  WFrag<T> qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) qf[kk] = window_row<T, HD, VEC>(Q + (long)min(myq, T_ - 1) * d, kk * 16 + 8 * g, d);
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();
  float m = -INFINITY, lsum = 0.0f;

  const KeyTiles<WA_BM, BN> kt(q0, T_, a.W, a.S);
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
    f32x16 s[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) s[h] = zero16();
    // consecutive products go to different halves' scores
    ahead<NH * NKK, AHEAD>([&](int i) { return Tile::row(sk, i % NH * 32 + li, i / NH * 16 + 8 * g); },
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
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
      m = mnew;
    }
    const float mns = m == -INFINITY ? 0.0f : m * a.scale_log2;
    float rs = 0.0f;
    WFrag<T> pf[2 * NH];
#pragma unroll
    for (int kc = 0; kc < 2 * NH; ++kc)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int r = 8 * (kc & 1) + e;
        rs = pf[kc].set2(e, fast_exp2(fmaf(s[kc >> 1][r], a.scale_log2, -mns)),
                         fast_exp2(fmaf(s[kc >> 1][r + 1], a.scale_log2, -mns)), rs);
      }
    lsum += rs + __shfl_xor(rs, 32);
    ahead<2 * NH * NDT, AHEAD>([&](int i) { return Tile::trans(sv, 16 * (i / NDT), i % NDT, l); },
                               [&](int i, const WFrag<T>& f) { o[i % NDT] = WFrag<T>::mma(f, pf[i / NDT], o[i % NDT]); });
  };
  auto advance = [&](int t) {  // the next tile into the other buffer, the one after it into registers
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
    if ((k0 <= qw + 31 && k0 + BN + a.W > qw + 1) || k0 < a.S) tile(t, std::true_type{});  // some pair is visible
    advance(t);
  }
  for (; t < kt.count; ++t) {
    tile(t, std::false_type{});
    advance(t);
  }

  if (myq >= T_) return;
  const float inv = 1.0f / lsum;
  T* O = (T*)a.out + (bh * T_ + myq) * d;
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
  if (g == 0 && a.lse != nullptr) a.lse[bh * T_ + myq] = (m * a.scale_log2 + __log2f(lsum)) * LN2;
}

// bf16 at head_dim 128: the same decomposition with tiles moved by 16-byte DMA loads into half-row-block LDS
// tiles (stage_hb: no staging registers, fragment addresses are bases plus immediates), two workgroups per CU,
// and K one tile ahead of V: the matrix products of the next tile's scores run between the exponentials of the
// current one wherever both are whole.
__global__ __launch_bounds__(256, 2) void window_fwd128_kernel(WindowArgs a) {
  constexpr int HD = 128, BN = 64, NKK = HD / 16, NDT = HD / 32;
  // X0 = {K buffer 0, V buffer 1}, X1 = {K buffer 1, V buffer 0}: iteration t (parity B) writes only X_B
  __shared__ __attribute__((aligned(16))) bf16 sX0[2 * BN * HD];
  __shared__ __attribute__((aligned(16))) bf16 sX1[2 * BN * HD];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T = a.T;
  const int q0 = (a.nx - 1 - xb) * WA_BM, qw = q0 + 32 * w, myq = qw + li;
  const bf16* Qrow = (const bf16*)a.q + (bh * T + min(myq, T - 1)) * HD;
  const long kvbase = bh / a.G * T * HD;
  // per-head buffer resources: rows past the end read as zeros (their scores are masked)
  const rsrc_t rK = make_rsrc((const bf16*)a.k + kvbase, (unsigned)T * HD * 2);
  const rsrc_t rV = make_rsrc((const bf16*)a.v + kvbase, (unsigned)T * HD * 2);

  bf16x8 qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) qf[kk] = *(const bf16x8*)(Qrow + kk * 16 + 8 * g);
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();
  float m = -INFINITY, lsum = 0.0f;

  const int grp = l >> 4, i16 = l & 15;
  const int d0 = 16 * (grp & 1) + 4 * (i16 & 3), kr = 4 * (grp >> 1) + (i16 >> 2);
  const int krow[2] = {hb_row_base(li, g, 0), hb_row_base(li, g, 1)};
  const int vtr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  const KeyTiles<WA_BM, BN> kt(q0, T, a.W, a.S);
  const int nkt = kt.count, whole = in_vector_register(kt.first_whole);
  auto visible = [&](int t) __attribute__((always_inline)) {
    const int k0 = kt.key0(t);
    return (k0 <= qw + 31 && k0 + BN + a.W > qw + 1) || k0 < a.S;
  };
  auto issue_k = [&](auto bt, int t) __attribute__((always_inline)) {
    stage_hb<BN>(rK, decltype(bt)::value ? sX1 : sX0, kt.key0(t), wu, l);
  };
  auto issue_v = [&](auto bt, int t) __attribute__((always_inline)) {
    stage_hb<BN>(rV, (decltype(bt)::value ? sX0 : sX1) + BN * HD, kt.key0(t), wu, l);
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
    const SeesKey sees(myq, kt.key0(t) + 4 * g, a.W, a.S);
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
  auto softmax_pair = [&](f32x16* s, int j, float mns, float& rs, bf16x8* pf, auto pin) __attribute__((always_inline)) {
    const int h = j >> 3, r = (2 * j) & 15;
    const float p0 = fast_exp2(fmaf(s[h][r], a.scale_log2, -mns)), p1 = fast_exp2(fmaf(s[h][r + 1], a.scale_log2, -mns));
    unsigned pk = pack_bf16x2(p0, p1);
    // the row sum of the bf16 P that the product consumes, one dot2 per pair
    rs = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk), bf16x2{(bf16)1.0f, (bf16)1.0f}, rs, false);
    if constexpr (decltype(pin)::value) asm volatile("" : "+v"(pk), "+v"(rs));
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
    float rs = 0.0f;
    bf16x8 pf[4];
#pragma unroll
    for (int j = 0; j < 16; ++j) softmax_pair(s, j, mns, rs, pf, std::false_type{});
    lsum += rs + __shfl_xor(rs, 32);
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
      softmax_pair(sc, i, mns, rs, pf, std::true_type{});
      __builtin_amdgcn_sched_barrier(0);
    }
    lsum += rs + __shfl_xor(rs, 32);
    pv_mma(bt, pf);
  };
  const std::integral_constant<int, 0> b0{};
  const std::integral_constant<int, 1> b1{};
  issue_k(b0, 0);
  issue_v(b0, 0);
  wait_vm();
  if (nkt > 1) issue_k(b1, 1);
  __syncthreads();  // K(0), V(0) visible
  if (visible(0)) scores(b0, sc);
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

  // O through the free array X0 (each wave its 32 rows), written as whole rows
  bf16* so = sX0 + w * 32 * HD;
  const float inv = myq < T ? 1.0f / lsum : 0.0f;
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
    if (qw + row < T)
      *(bf16x8*)((bf16*)a.out + (bh * T + qw + row) * HD + 8 * ch) = *(const bf16x8*)(so + lds_off<HD>(row, 8 * ch));
  }
  if (myq < T && g == 0 && a.lse != nullptr) a.lse[bh * T + myq] = (m * a.scale_log2 + __log2f(lsum)) * LN2;
}

template <typename T, int BN, bool VEC>
void launch_fwd(hipStream_t s, WindowArgs a, int BH) {
  a.nx = (a.T + WA_BM - 1) / WA_BM;
  const unsigned grid = (unsigned)a.nx * (unsigned)BH;
  if constexpr (sizeof(T) == 2 && VEC) {
    if (a.d == 128) {
      window_fwd128_kernel<<<grid, 256, 0, s>>>(a);
      return;
    }
  }
  if (a.d <= 32)
    window_fwd_kernel<T, 32, BN, VEC><<<grid, 256, 0, s>>>(a);
  else if (a.d <= 64)
    window_fwd_kernel<T, 64, BN, VEC><<<grid, 256, 0, s>>>(a);
  else if (a.d <= 96)
    window_fwd_kernel<T, 96, BN, VEC><<<grid, 256, 0, s>>>(a);
  else
    window_fwd_kernel<T, 128, BN, VEC><<<grid, 256, 0, s>>>(a);
}

}  // namespace

int window_check(int batch, int num_heads, int num_kv_heads, int seq_len, int head_dim, int window, int sinks,
                 int dtype) {
  EDF_REQUIRE(batch > 0 && num_heads > 0 && num_kv_heads > 0 && seq_len > 0 && head_dim > 0, EDF_ERR_INVALID_ARG,
              "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(num_heads % num_kv_heads == 0, EDF_ERR_INVALID_ARG, "num_heads %d is no multiple of num_kv_heads %d",
              num_heads, num_kv_heads);
  EDF_REQUIRE(window > 0 && sinks >= 0, EDF_ERR_INVALID_ARG, "window must be positive and sinks not negative");
  EDF_REQUIRE(sinks <= (1 << 22), EDF_ERR_UNSUPPORTED, "sinks must be at most 2^22");
  EDF_REQUIRE(head_dim <= 128, EDF_ERR_UNSUPPORTED, "head_dim %d > 128 unsupported", head_dim);
  EDF_REQUIRE(seq_len < (1 << 30) && (long)batch * num_heads < (1L << 31) &&
                  (double)batch * num_heads * ((seq_len + 31) / 32) < 2147483648.0,
              EDF_ERR_UNSUPPORTED, "batch x heads x seq_len too large for one call");
  return EDF_OK;
}

}  // namespace edf

extern "C" {

int edf_window_attention(void* stream, const void* q, const void* k, const void* v, void* out, float* lse, int batch,
                         int num_heads, int num_kv_heads, int seq_len, int head_dim, int window, int sinks,
                         int dtype) {
  using namespace edf;
  const int rc = window_check(batch, num_heads, num_kv_heads, seq_len, head_dim, window, sinks, dtype);
  if (rc) return rc;
  EDF_REQUIRE(q && k && v && out, EDF_ERR_INVALID_ARG, "null tensor pointer");
  WindowArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = out, a.lse = lse;
  a.T = seq_len, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window < seq_len ? window : seq_len, a.S = sinks < seq_len ? sinks : seq_len;
  a.scale = 1.0f / sqrtf((float)head_dim), a.scale_log2 = a.scale * LOG2E;
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out;
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15) && seq_len <= WINDOW_VEC_T;
  hipStream_t s = as_stream(stream);
  const int BH = batch * num_heads;
  if (window_narrow(BH, seq_len, vec)) return window_narrow_run(false, s, a, BH, dtype);
  if (dtype == EDF_BF16)
    vec ? launch_fwd<bf16, 64, true>(s, a, BH) : launch_fwd<bf16, 64, false>(s, a, BH);
  else
    vec ? launch_fwd<float, 32, true>(s, a, BH) : launch_fwd<float, 32, false>(s, a, BH);
  return check_launch("window attention");
}

}  // extern "C"
