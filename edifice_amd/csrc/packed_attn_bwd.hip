// Causal attention over texts laid end to end, backward (packed_attn.hip has the forward and its formulas):
//   P from the forward's row sums; dV_j = sum_i P_ij dO_i, dP = dO V^T, D_i = dO_i . O_i,
//   dS = P (dP - D) / sqrt(d), dQ = dS K, dK = dS^T Q; dK, dV summed over the query heads of a key head.
// 10 d flops per visible pair (S and dP formed twice, once for each kernel): bound by the matrix cores.
//
//   dQ: a workgroup's four waves own 32 queries each (Q^T and dO^T in registers) and walk the key tiles of the forward; it
//   also forms D and leaves it for the second kernel.
//   dK, dV: a workgroup owns 128 keys of a text (32 per wave, K^T and V^T in registers) of one key head and walks the
//   query tiles that see one of them, query head by query head: the sum over shared heads needs no atomics.  Where key
//   blocks are few against the GPU, their query tiles are cut into chunks, as those of the queries are, which leave float32
//   sums, added in order by a third kernel.
// 12 texts to 4096, 32(8)x128, bf16: dQ 853 us (947 TFLOP/s of the 6 d that it does), dK and dV 1210 (890 of 8 d), profiled.
// 5 texts to 700, 8(4)x64, float32: 25 + 31 us, and 4 + 6 for the sums of chunks.
// In bf16 P and dS are rounded as operands of the second products (2^-8 of each term); D is formed from the rounded O that
// the forward left, or where keys are few, and O with its rounding as large as V, as sum P dP; everything else is float32.
// (O's rounding kept in bf16 beside it does the same for twice the bytes of O: forward and backward of 200 texts of 150
// tokens on average, 16(4)x64, 296 us, and 260 so; of 60 texts of 300, 16(4)x128, 392 and 334.)
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "edf_packed.hpp"

namespace edf {
namespace {

template <typename T, int HD, int BN, bool VEC>
__global__ __launch_bounds__(256, 1) void packed_dq_kernel(PackArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32, NH = BN / 32;
  constexpr int AHEAD = sizeof(T) == 2 ? 3 : 1;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, l = tid & 63, g = l >> 5, li = l & 31;
  const QueryTile<BN> qt(a, sK);
  if (qt.none) return;
  const int d = a.d, myq = qt.myq, myp = qt.pw + li;
  const long qrow = qt.row0 + min(myq, qt.nq - 1);
  const T *K = (const T*)a.k + qt.krow * d, *V = (const T*)a.v + qt.krow * d;

  // With few keys O is as large as V, and its rounding shows in D = dO . O: D = sum P dP there, from the tiles themselves
  // (all of them: a chunk has four tiles at least).
  const bool few = sizeof(T) == 2 && qt.kt.count <= 2;
  WFrag<T> qf[NKK], of[NKK];
  float dd = 0.0f;
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const int col = kk * 16 + 8 * g;
    qf[kk] = window_row<T, HD, VEC>((const T*)a.q + qrow * d, col, d);
    of[kk] = window_row<T, HD, VEC>((const T*)a.go + qrow * d, col, d);
  }
  if (!few) {
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const WFrag<T> oo = window_row<T, HD, VEC>((const T*)a.o + qrow * d, kk * 16 + 8 * g, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) dd = fmaf(oo.get(e), of[kk].get(e), dd);
    }
    dd += __shfl_xor(dd, 32);
  }
  const float lse = a.lse[qrow] * LOG2E;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zero16();

  const int count = qt.t1 - qt.t0;
  const TileLoader<T, HD, BN, VEC> ld(tid, d, qt.nk);
  WFrag<T> rk[ld.N], rv[ld.N];
  auto gload = [&](int t) {
    const int k0 = qt.key0(t);
    ld.load(K, k0, rk);
    ld.load(V, k0, rv);
  };
  auto sstore = [&](int buf) {
    ld.template store<Tile>(sK[buf], rk);
    ld.template store<Tile>(sV[buf], rv);
  };
  auto scores = [&](int t, f32x16* s, f32x16* dp) {
    const T *sk = sK[t & 1], *sv = sV[t & 1];
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
  };
  auto row_sum = [&](int t) {  // this lane's share of sum P dP
    const SeesKey sees(myp, qt.key0(t) + 4 * g, a.W, a.sinks);
    f32x16 s[NH], dp[NH];
    scores(t, s, dp);
    float x = 0.0f;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float y = fast_exp2(fmaf(s[h][r], a.scale_log2, -lse)) * dp[h][r];
        x += sees(h * 32 + d_row(r, 0)) ? y : 0.0f;
      }
    return x;
  };
  auto tile = [&](int t, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const SeesKey sees(myp, qt.key0(t) + 4 * g, a.W, a.sinks);
    const T* sk = sK[t & 1];
    f32x16 s[NH], dp[NH];
    scores(t, s, dp);
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
  if (few) {  // both tiles at once, gone through twice
    if (count > 1) sstore(1);
    __syncthreads();
    for (int t = 0; t < count; ++t)
      if (qt.visible(a, qt.key0(t), BN)) dd += row_sum(t);
    dd += __shfl_xor(dd, 32);
    for (int t = 0; t < count; ++t)
      if (qt.visible(a, qt.key0(t), BN)) tile(t, std::true_type{});
  } else {
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
  }
  if (g == 0 && myq < qt.nq && qt.first) a.dd[qrow] = dd;
  if (myq >= qt.nq) return;
  if (qt.slot >= 0) {
    float* out = a.part + qt.slot * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) =
            f32x4{dq[dt][rb * 4], dq[dt][rb * 4 + 1], dq[dt][rb * 4 + 2], dq[dt][rb * 4 + 3]};
    return;
  }
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
__global__ __launch_bounds__(256, 2) void packed_dq128_kernel(PackArgs a) {
  constexpr int HD = 128, BN = 64, NKK = HD / 16, NDT = HD / 32;
  __shared__ __attribute__((aligned(16))) bf16 sR0[2 * BN * HD];  // ring slot: K then V
  __shared__ __attribute__((aligned(16))) bf16 sR1[2 * BN * HD];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  const QueryTile<BN> qt(a, sR0);
  if (qt.none) return;
  const int pw = qt.pw, myp = pw + li, myq = qt.myq;
  const long qrow = qt.row0 + min(myq, qt.nq - 1);
  const rsrc_t rK = make_rsrc((const bf16*)a.k + qt.krow * HD, (unsigned)qt.nk * HD * 2);
  const rsrc_t rV = make_rsrc((const bf16*)a.v + qt.krow * HD, (unsigned)qt.nk * HD * 2);

  const bool few = qt.kt.count <= 2;  // as above
  bf16x8 qf[NKK], of[NKK];
  float dd = 0.0f;
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const long at = qrow * HD + kk * 16 + 8 * g;
    qf[kk] = *(const bf16x8*)((const bf16*)a.q + at);
    of[kk] = *(const bf16x8*)((const bf16*)a.go + at);
  }
  if (!few) {
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const bf16x8 ov = *(const bf16x8*)((const bf16*)a.o + qrow * HD + kk * 16 + 8 * g);
#pragma unroll
      for (int e = 0; e < 8; ++e) dd = fmaf((float)of[kk][e], (float)ov[e], dd);
    }
    dd += __shfl_xor(dd, 32);
  }
  const float lse = a.lse[qrow] * LOG2E;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zero16();

  const int grp = l >> 4, i16 = l & 15;
  const int d0 = 16 * (grp & 1) + 4 * (i16 & 3), kr = 4 * (grp >> 1) + (i16 >> 2);
  const int krow[2] = {hb_row_base(li, g, 0), hb_row_base(li, g, 1)};
  const int ktr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  const int count = qt.t1 - qt.t0, whole = in_vector_register(max(qt.kt.first_whole - qt.t0, 0));
  auto issue = [&](auto bt, int t) {
    constexpr int B = decltype(bt)::value;
    const int k0 = qt.key0(t);
    stage_hb<BN>(rK, B ? sR1 : sR0, k0, wu, l);
    stage_hb<BN>(rV, (B ? sR1 : sR0) + BN * HD, k0, wu, l);
  };
  // S and dP of the 32 keys of half h (a constant) of a tile
  auto scores = [&](const bf16* sK, int h, f32x16& s, f32x16& dp) __attribute__((always_inline)) {
    const bf16* sV = sK + BN * HD;
    s = zero16();
    dp = zero16();
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int off = krow[kk & 1] + hb_row_off<BN>(kk, 32 * h);
      s = mfma32(*(const bf16x8*)(&sK[off]), qf[kk], s);
      dp = mfma32(*(const bf16x8*)(&sV[off]), of[kk], dp);
    }
  };
  auto row_sum = [&](auto bt, int t) {  // this lane's share of sum P dP
    const bf16* sK = decltype(bt)::value ? sR1 : sR0;
    const int k0 = qt.key0(t);
    float x = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kb = k0 + 32 * h;
      if (!qt.visible(a, kb, 32)) continue;
      const SeesKey sees(myp, kb + 4 * g, a.W, a.sinks);
      f32x16 s, dp;
      scores(sK, h, s, dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float y = fast_exp2(fmaf(s[r], a.scale_log2, -lse)) * dp[r];
        x += sees(d_row(r, 0)) ? y : 0.0f;
      }
    }
    return x;
  };
  auto tile = [&](auto bt, int t, auto masked) {
    constexpr bool MASK = decltype(masked)::value;
    const bf16* sK = decltype(bt)::value ? sR1 : sR0;
    const int k0 = qt.key0(t);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kb = k0 + 32 * h;
      if (MASK && !qt.visible(a, kb, 32)) continue;  // no visible pair
      const SeesKey sees(myp, kb + 4 * g, a.W, a.sinks);
      f32x16 s, dp;
      scores(sK, h, s, dp);
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
    if (t + 1 < count) issue(ot, t + 1);
    if (t >= whole) tile(bt, t, std::false_type{});
    else tile(bt, t, std::true_type{});
    wait_vm();
    __syncthreads();
  };
  const std::integral_constant<int, 0> b0{};
  const std::integral_constant<int, 1> b1{};
  if (count > 0) issue(b0, 0);
  if (few && count > 1) issue(b1, 1);
  wait_vm();
  __syncthreads();
  if (few) {  // both tiles at once, gone through twice
    if (count > 0) dd = row_sum(b0, 0);
    if (count > 1) dd += row_sum(b1, 1);
    dd += __shfl_xor(dd, 32);
    if (count > 0) tile(b0, 0, std::true_type{});
    if (count > 1) tile(b1, 1, std::true_type{});
  } else {
    for (int t = 0; t < count; t += 2) {
      step(b0, t);
      if (t + 1 < count) step(b1, t + 1);
    }
  }
  if (g == 0 && myq < qt.nq && qt.first) a.dd[qrow] = dd;
  if (myq >= qt.nq) return;
  if (qt.slot >= 0) {
    float* out = a.part + qt.slot * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) =
            f32x4{dq[dt][rb * 4], dq[dt][rb * 4 + 1], dq[dt][rb * 4 + 2], dq[dt][rb * 4 + 3]};
    return;
  }
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

// The (query head, tile of BQ queries) pairs that a block of keys from row `first` of n on walks, in a text of m queries: nt
// tiles a head, from query qs on.
template <int BQ>
struct QueryTiles {
  int qs, nt;
  EDF_DEVICE QueryTiles(const PackArgs& a, int first, int n, int m) {
    const int ahead = n - m;
    qs = max(0, first - ahead);  // the first query that sees the block's first key
    int end = m;
    if (first >= a.sinks) end = (int)min((long)m, (long)first + PK_M - 1 + a.W - ahead);  // past the last key's window
    nt = max(0, (end - qs + BQ - 1) / BQ);
  }
};

// The key block of a dK, dV workgroup and its chunk [t0, t1) of the block's pairs; LEAST: of a chunk.
template <int BQ, int LEAST>
struct KeyBlock {
  int head, krow, nk, first, qrow, nq, qs, nt, t0, t1;  // first: the block's first key within the text
  long slot;                                            // of one of several chunks: its place in part, or -1
  bool none;
  EDF_DEVICE int ahead() const { return nk - nq; }
  // the first query of pairs i G .. (i + 1) G - 1: from a text's end backwards, so that the blocks that are under way meet in
  // the same queries (12 texts to 4096, 32(8)x128, and 8 to 2000, 8(4)x64: 1 to 2% of forward and backward)
  EDF_DEVICE int query(int i) const { return qs + (nt - 1 - i) * BQ; }
  // lds: 5 KB that the kernel uses later
  EDF_DEVICE KeyBlock(const PackArgs& a, void* lds) : slot(-1) {
    const int hkv = a.H / a.G;
    int x, chunk = 0, len = 0;
    none = !packed_block(hkv, a.items > 0 ? a.items : a.nx, x, head);
    if (none) return;
    TextTile t;
    if (a.items > 0) {
      const Item it = find_item(a.ko, a.M, a.qo, a.N, a.S, 7, hkv, LEAST, x, (int*)lds,
                                [&](int first, int n, int m) { return QueryTiles<BQ>(a, first, n, m).nt * a.G; });
      none = it.none;
      if (none) return;
      t = it.tile, chunk = it.chunk, len = it.len;
      if (it.chunks > 1) slot = (long)head * a.items + x;
      if (chunk == 0 && threadIdx.x == 0) {
        int* p = a.plan + 2 * ((long)head * a.nx + it.x);
        p[0] = x;
        p[1] = it.chunks;
      }
    } else {
      t = a.by_work ? find_tile_by_work(a.ko, a.M, a.qo, a.N, a.S, 7, x, false)
                    : find_tile(a.ko, a.M, a.qo, a.N, a.S, 7, x);
      none = t.first >= t.n;
      if (none) return;
    }
    krow = t.row0, nk = t.n, first = t.first;
    qrow = t.other0, nq = t.m;
    const QueryTiles<BQ> q(a, first, nk, nq);
    qs = q.qs, nt = q.nt;
    t0 = chunk * len;
    t1 = a.items > 0 ? min(t0 + len, nt * a.G) : nt * a.G;
  }
};

// Two workgroups a CU in bf16 up to 96 elements a head (at 96, 17 registers are spilled for it); elsewhere the two
// accumulators and the fragments of K and V want more than 256 registers.
template <typename T, int HD, int BQ, bool VEC>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && HD <= 96 && VEC ? 2 : 1)) void packed_dkdv_kernel(PackArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  constexpr int AHEAD = sizeof(T) == 4 ? 1 : HD == 96 ? 2 : 3;
  using Tile = WTile<T, HD, BQ>;
  __shared__ __attribute__((aligned(16))) T sQ[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sO[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) float sL[2][BQ], sD[2][BQ];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const KeyBlock<BQ, sizeof(T) == 2 ? 2 : 1> kb(a, sQ);
  if (kb.none) return;
  const int head = kb.head;
  const int d = a.d, kw = kb.first + 32 * w, mykey = kw + li, t0 = kb.t0, t1 = kb.t1;
  const long krow = (long)head * a.M + kb.krow + min(mykey, kb.nk - 1);
  WFrag<T> kf[NKK], vf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    kf[kk] = window_row<T, HD, VEC>((const T*)a.k + krow * d, kk * 16 + 8 * g, d);
    vf[kk] = window_row<T, HD, VEC>((const T*)a.v + krow * d, kk * 16 + 8 * g, d);
  }
  f32x16 dk[NDT], dv[NDT];  // dK^T, dV^T: rows are dims, the column this lane's key
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    dk[dt] = zero16();
    dv[dt] = zero16();
  }
  const TileLoader<T, HD, BQ, VEC> ld(tid, d, kb.nq);
  WFrag<T> rq[ld.N], ro[ld.N];
  float rl = 0.0f, rd = 0.0f;
  auto gload = [&](int t) {
    const int i = t / a.G, h = t - i * a.G, q0 = kb.query(i);
    const long base = (long)(head * a.G + h) * a.N + kb.qrow;
    ld.load((const T*)a.q + base * d, q0, rq);
    ld.load((const T*)a.go + base * d, q0, ro);
    if (tid < BQ) {
      const long q = base + min(q0 + tid, kb.nq - 1);
      rl = q0 + tid < kb.nq ? a.lse[q] * LOG2E : INFINITY;  // a query past the end gets P = 0
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
    const int p0 = kb.query(t / a.G) + kb.ahead();  // position of the tile's first query
#pragma unroll
    for (int sub = 0; sub < BQ / 32; ++sub) {
      const int pb = p0 + 32 * sub;
      // no query of the sub-tile sees a key of this wave
      if (pb + 31 < kw || (pb > kw + 30 + a.W && kw >= a.sinks)) continue;
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
              const bool see = window_sees(pb + 8 * rb + 4 * g + e, mykey, a.W, a.sinks);
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
      if (pb >= kw + 31 && pb + 31 - kw < a.W) subtile(std::false_type{});
      else subtile(std::true_type{});
    }
    if (t + 1 < t1) {
      sstore(buf ^ 1);
      if (t + 2 < t1) gload(t + 2);
    }
    __syncthreads();
  }
  if (mykey >= kb.nk) return;
  if (kb.slot >= 0) {  // these sums are of a chunk: [key head][item][dK | dV][key][dim]
    float* out = a.part + kb.slot * (2L * PK_M * HD) + (32 * w + li) * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        f32x4 u, v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = dk[dt][rb * 4 + e];
          v[e] = dv[dt][rb * 4 + e];
        }
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) = u;
        *(f32x4*)(out + PK_M * HD + dt * 32 + 8 * rb + 4 * g) = v;
      }
    return;
  }
  T *kout = (T*)a.dk + krow * d, *vout = (T*)a.dv + krow * d;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int c = dt * 32 + 8 * rb + 4 * g;
      if (VEC && c + 4 <= d) {
        typedef __attribute__((ext_vector_type(4))) T vec4;
        vec4 u, v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = from_f32<T>(dk[dt][rb * 4 + e] * a.scale);
          v[e] = from_f32<T>(dv[dt][rb * 4 + e]);
        }
        *(vec4*)(kout + c) = u;
        *(vec4*)(vout + c) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < d) {
            kout[c + e] = from_f32<T>(dk[dt][rb * 4 + e] * a.scale);
            vout[c + e] = from_f32<T>(dv[dt][rb * 4 + e]);
          }
      }
    }
}

// dK, dV, bf16 at head_dim 128: V is read from an LDS copy of the workgroup's 128 keys (its fragments would not
// fit 256 registers beside the two accumulators), Q and dO come in 32-query tiles by DMA loads, two workgroups per
// CU.
__global__ __launch_bounds__(256, 2) void packed_dkdv128_kernel(PackArgs a) {
  constexpr int HD = 128, BQ = 32, NKK = HD / 16, NDT = HD / 32;
  __shared__ __attribute__((aligned(16))) bf16 sV[PK_M * HD];
  __shared__ __attribute__((aligned(16))) bf16 sR0[2 * BQ * HD];  // ring slot: Q then dO
  __shared__ __attribute__((aligned(16))) bf16 sR1[2 * BQ * HD];
  __shared__ __attribute__((aligned(16))) float sL0[BQ], sL1[BQ], sD0[BQ], sD1[BQ];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  const KeyBlock<BQ, 2> kb(a, sR0);
  if (kb.none) return;
  const int head = kb.head;
  const int kw = kb.first + 32 * w, mykey = kw + li, t0 = kb.t0, t1 = kb.t1;
  const long kbase = (long)head * a.M + kb.krow, krow = kbase + min(mykey, kb.nk - 1);

  // keys past the text's end read zero rows of V: they only feed their own columns, never stored
  stage_hb<PK_M>(make_rsrc((const bf16*)a.v + kbase * HD, (unsigned)kb.nk * HD * 2), sV, kb.first, wu, l);
  bf16x8 kf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk)
    kf[kk] = *(const bf16x8*)((const bf16*)a.k + krow * HD + kk * 16 + 8 * g);
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
    const int i = t / a.G, h = t - i * a.G, q0 = kb.query(i);
    const long row = (long)(head * a.G + h) * a.N + kb.qrow;
    stage_hb<BQ>(make_rsrc((const bf16*)a.q + row * HD, (unsigned)kb.nq * HD * 2), B ? sR1 : sR0, q0, wu, l);
    stage_hb<BQ>(make_rsrc((const bf16*)a.go + row * HD, (unsigned)kb.nq * HD * 2), (B ? sR1 : sR0) + BQ * HD, q0, wu, l);
    if (tid < BQ) {
      const long q = row + min(q0 + tid, kb.nq - 1);
      rl = q0 + tid < kb.nq ? a.lse[q] : INFINITY;  // a query past the end gets P = 0
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
  const int vrow[2] = {hb_row_base(li, g, 0) + hb_row_off<PK_M>(0, 32 * w),
                       hb_row_base(li, g, 1) + hb_row_off<PK_M>(0, 32 * w)};
  const int qtr[2] = {hb_tr_base(kr, d0, 0), hb_tr_base(kr, d0, 1)};
  auto subtile = [&](auto bt, int pb, auto masked) {
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
      const bf16x8 vf = *(const bf16x8*)(&sV[vrow[kk & 1] + hb_row_off<PK_M>(kk, 0)]);
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
          const bool see = window_sees(pb + 8 * rb + 4 * g + e, mykey, a.W, a.sinks);
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
    const int pb = kb.query(t / a.G) + kb.ahead();  // position of the tile's first query
    if (!(pb + 31 < kw || (pb > kw + 30 + a.W && kw >= a.sinks))) {  // some query sees a key of this wave
      if (pb >= kw + 31 && pb + 31 - kw < a.W) subtile(bt, pb, std::false_type{});
      else subtile(bt, pb, std::true_type{});
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
  if (mykey >= kb.nk) return;
  if (kb.slot >= 0) {  // these sums are of a chunk: [key head][item][dK | dV][key][dim]
    float* out = a.part + kb.slot * (2L * PK_M * HD) + (32 * w + li) * HD;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb) {
        f32x4 u, v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = dk[dt][rb * 4 + e];
          v[e] = dv[dt][rb * 4 + e];
        }
        *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) = u;
        *(f32x4*)(out + PK_M * HD + dt * 32 + 8 * rb + 4 * g) = v;
      }
    return;
  }
  const long row = krow * HD;
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

// dK, dV of blocks whose query tiles are in chunks, added in order, four elements a thread.  A workgroup takes one of the
// pieces of a block's [dK | dV][key][dim].
template <typename T, int HD>
__global__ __launch_bounds__(256) void packed_sum_kernel(PackArgs a) {
  constexpr int PIECES = 2 * PK_M * HD / 1024;
  const int piece = blockIdx.x % PIECES, x = blockIdx.x / PIECES % a.nx, head = blockIdx.x / PIECES / a.nx;
  const TextTile t = find_tile(a.ko, a.M, a.qo, a.N, a.S, 7, x);
  const int e = (piece * 256 + threadIdx.x) * 4;
  const bool is_v = e >= PK_M * HD;
  const int key = t.first + e / HD % PK_M, c = e % HD;
  if (t.first >= t.n || key >= t.n || c >= a.d) return;
  const int* p = a.plan + 2 * ((long)head * a.nx + x);
  const int item = p[0], n = p[1];
  if (n <= 1 || item < 0 || n > a.items - item) return;  // one chunk, or no plan (offsets that do not ascend)
  const float* in = a.part + ((long)head * a.items + item) * (2L * PK_M * HD) + e;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = 0; i < n; ++i) s += *(const f32x4*)(in + i * (2L * PK_M * HD));
  if (!is_v) s *= a.scale;
  T* out = (T*)(is_v ? a.dv : a.dk) + ((long)head * a.M + t.row0 + key) * a.d + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < a.d) out[i] = from_f32<T>(s[i]);
}

// dQ of rows whose key tiles are in chunks, added in order, four elements a lane.
template <typename T, int HD>
__global__ __launch_bounds__(256) void packed_dq_sum_kernel(PackArgs a) {
  constexpr int LANES = HD <= 32 ? 8 : HD <= 64 ? 16 : 32;
  const ChunkRow<LANES> r(a);
  const int e = 4 * (threadIdx.x % LANES);
  if (r.chunks == 0 || e >= a.d) return;
  const float* in = a.part + r.slot * HD + e;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int c = 0; c < r.chunks; ++c) s += *(const f32x4*)(in + (long)PK_M * HD * c);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < a.d) st((T*)a.dq, r.row * a.d + e + i, s[i] * a.scale);
}

constexpr int BQ_BF16 = 64, BQ_32 = 32;  // query tiles of dK, dV: bf16, and float32

// Key blocks a head, and whether and into how many chunks their query tiles are cut: where the blocks would not fill the
// GPU's 512 places, and query tiles are enough that chunks are worth the kernel that adds them.
void backward_plan(PackArgs& a, int dtype) {
  a.nx = (int)packed_tiles(a.M, a.S, PK_M);
  const long hkv = a.H / a.G, wgs = hkv * a.nx, queries = (long)a.N * a.G;
  a.by_work = order_by_work(a, wgs);
  // (the plan's sum of tiles is an int)
  const bool cut = wgs < PK_PLAN && queries > (dtype == EDF_BF16 ? 512 : 64) && queries < (1 << 25) && a.M < (1 << 24);
  a.items = cut ? (int)((PK_ITEMS + hkv - 1) / hkv) + a.nx : 0;
}
size_t key_bytes(const PackArgs& a) {
  const size_t hkv = a.H / a.G;
  return a.items == 0 ? 0 : hkv * a.items * (2 * PK_M) * window_pad(a.d) * sizeof(float) + hkv * a.nx * 2 * sizeof(int);
}
// the larger of what the two kernels leave, one after the other
size_t part_bytes(PackArgs a, int dtype) {
  query_plan(a, key_tile(dtype));
  const size_t queries = chunk_bytes(a, 0);
  backward_plan(a, dtype);
  return std::max(queries, key_bytes(a));
}
size_t row_bytes(long heads, long rows) { return ((size_t)heads * rows * sizeof(float) + 255) & ~(size_t)255; }

template <typename T, int HD, int BN, int BQ, bool VEC>
int launch_bwd(hipStream_t s, PackArgs a) {
  constexpr bool dma = sizeof(T) == 2 && HD == 128 && VEC;
  const bool fast = dma && a.d == 128;
  PackArgs q = a;
  query_plan(q, BN);
  chunk_memory(q, a.part, 0);
  const long groups = a.H >> q.hs;
  const unsigned qgrid = (unsigned)packed_grid(groups, q.items > 0 ? q.items : q.nx);
  const int hkv = a.H / a.G;
  const unsigned kgrid = (unsigned)packed_grid(hkv, a.items > 0 ? a.items : a.nx);
  if (fast) packed_dq128_kernel<<<qgrid, 256, 0, s>>>(q);
  else packed_dq_kernel<T, HD, BN, VEC><<<qgrid, 256, 0, s>>>(q);
  int rc = check_launch("packed attention dQ");
  if (rc) return rc;
  if (q.items > 0) {
    packed_dq_sum_kernel<T, HD>
        <<<(unsigned)packed_grid(groups, (long)q.nx * (HD <= 32 ? 4 : HD <= 64 ? 8 : 16)), 256, 0, s>>>(q);
    rc = check_launch("packed attention dQ sums");
    if (rc) return rc;
  }
  if (fast) packed_dkdv128_kernel<<<kgrid, 256, 0, s>>>(a);
  else packed_dkdv_kernel<T, HD, BQ, VEC><<<kgrid, 256, 0, s>>>(a);
  rc = check_launch("packed attention dK, dV");
  if (rc || a.items == 0) return rc;
  packed_sum_kernel<T, HD><<<(unsigned)(2L * PK_M * HD / 1024 * a.nx * hkv), 256, 0, s>>>(a);
  return check_launch("packed attention dK, dV sums");
}
template <typename T, int BN, int BQ, bool VEC>
int launch_bwd_d(hipStream_t s, const PackArgs& a) {
  switch (window_pad(a.d)) {
    case 32: return launch_bwd<T, 32, BN, BQ, VEC>(s, a);
    case 64: return launch_bwd<T, 64, BN, BQ, VEC>(s, a);
    case 96: return launch_bwd<T, 96, BN, BQ, VEC>(s, a);
    default: return launch_bwd<T, 128, BN, BQ, VEC>(s, a);
  }
}

}  // namespace
}  // namespace edf

extern "C" {

size_t edf_packed_attention_backward_workspace_bytes(int num_heads, int num_kv_heads, long rows, long key_rows, int texts,
                                                     int head_dim, int window, int sinks, int dtype) {
  using namespace edf;
  if (packed_check(num_heads, num_kv_heads, rows, key_rows, texts, head_dim, window, sinks, dtype)) return 0;
  PackArgs a{};
  a.N = (int)rows, a.M = (int)key_rows, a.S = texts, a.H = num_heads, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window > 0 ? std::min(window, PK_ALL) : PK_ALL, a.sinks = sinks;
  return row_bytes(num_heads, rows) + part_bytes(a, dtype);
}

int edf_packed_attention_backward(void* stream, const void* q, const void* k, const void* v, const int32_t* offsets,
                                  const int32_t* key_offsets, const void* out, const void* grad_out, const float* lse,
                                  void* grad_q, void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes,
                                  int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim,
                                  int window, int sinks, int dtype) {
  using namespace edf;
  const int rc = packed_check(num_heads, num_kv_heads, rows, key_rows, texts, head_dim, window, sinks, dtype);
  if (rc) return rc;
  EDF_REQUIRE(q && k && v && offsets && key_offsets && out && grad_out && lse && grad_q && grad_k && grad_v,
              EDF_ERR_INVALID_ARG, "null tensor pointer (the forward's lse is required)");
  PackArgs a{};
  a.q = q, a.k = k, a.v = v, a.qo = offsets, a.ko = key_offsets, a.o = out, a.go = grad_out;
  a.lse = const_cast<float*>(lse), a.dq = grad_q, a.dk = grad_k, a.dv = grad_v;
  a.N = (int)rows, a.M = (int)key_rows, a.S = texts, a.H = num_heads, a.G = num_heads / num_kv_heads, a.d = head_dim;
  a.W = window > 0 ? std::min(window, PK_ALL) : PK_ALL, a.sinks = sinks;
  a.scale = 1.0f / sqrtf((float)head_dim), a.scale_log2 = a.scale * LOG2E;
  backward_plan(a, dtype);
  const size_t need = row_bytes(num_heads, rows) + part_bytes(a, dtype);
  EDF_REQUIRE(workspace && workspace_bytes >= need, EDF_ERR_WORKSPACE, "workspace too small: need %zu bytes", need);
  a.dd = (float*)workspace;
  a.part = (float*)((char*)workspace + row_bytes(num_heads, rows));
  a.plan = (int*)(a.part + (size_t)(a.H / a.G) * a.items * (2 * PK_M) * window_pad(a.d));
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)grad_out |
                         (uintptr_t)grad_q | (uintptr_t)grad_k | (uintptr_t)grad_v;
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15) &&
                   std::max(rows, key_rows) <= WINDOW_VEC_T;
  hipStream_t s = as_stream(stream);
  if (dtype == EDF_BF16)
    return vec ? launch_bwd_d<bf16, 64, BQ_BF16, true>(s, a) : launch_bwd_d<bf16, 64, BQ_BF16, false>(s, a);
  return vec ? launch_bwd_d<float, 32, BQ_32, true>(s, a) : launch_bwd_d<float, 32, BQ_32, false>(s, a);
}

}  // extern "C"
