// Attention with a sliding window and sinks (window_attn.hip has the formulas), narrow form of the forward and dQ:
// a workgroup owns 32 queries and its four waves divide the key tiles among them, each with results of its own that
// are joined in LDS at the end.  No tile is shared, so there is no barrier in the loops, and a call has four times
// the workgroups of the wide form: it takes the calls whose wide grid would leave the GPU half empty
// (window_narrow).  Rows of whole 16-byte pieces only.  The far queries' kernel at the end is built the same way.
//
// Row operands (a lane's 8 elements of one row) come straight from memory, a tile ahead of their use.
// Transposed operands come through a wave-private LDS copy of the tile; the forward in float32 past head_dim 64 reads
// V^T straight from memory (a 32-lane row piece is 128 contiguous bytes; 1x8(4)x1000x128 window 300: 24.9 us, 29.4 through
// LDS; at 64 27.1 and 25.8, and dQ 49.8 and 36.9 at 128).
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "edf_window.hpp"

namespace edf {
namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr int WN_R = 32, WN_WAVES = 4;  // rows per workgroup; waves

// The 32-row tile of a tensor [T, d] at row r0 as a wave reads it.
template <typename T, int HD, bool LDS>
struct NTile {
  static constexpr int NKK = HD / 16, NDT = HD / 32;
  using Tile = WTile<T, HD, WN_R>;
  // rows past the end repeat the last one: their scores are masked
  template <bool VEC = true>
  EDF_DEVICE static void rows(const T* x, int r0, int T_, int d, int l, WFrag<T>* f) {
    const T* row = x + (long)min(r0 + (l & 31), T_ - 1) * d;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) f[kk] = window_row<T, HD, VEC>(row, kk * 16 + 8 * (l >> 5), d);
  }
  EDF_DEVICE static void keep(T* lds, int l, const WFrag<T>* f) {  // row fragments into the wave's LDS tile
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) f[kk].store(lds + Tile::off(l & 31, kk * 16 + 8 * (l >> 5)));
  }
  // transposed operand: columns 32 dt + (lane % 32), rows 16 kc + {4 g .. + 3, 8 + 4 g .. + 3} of the tile
  EDF_DEVICE static WFrag<T> trans(const T* x, const T* lds, int r0, int T_, int d, int kc, int dt, int l) {
    if constexpr (LDS) {
      return Tile::trans(lds, 16 * kc, dt, l);
    } else {
      WFrag<T> f;
      const int c = min(dt * 32 + (l & 31), d - 1), r = r0 + 16 * kc + 4 * (l >> 5);
#pragma unroll
      for (int e = 0; e < 8; ++e) f.set(e, x[(long)min(r + (e < 4 ? e : e + 4), T_ - 1) * d + c]);
      return f;
    }
  }
};

// Sum of the four waves' accumulators into wave 0's, two halves at a time through LDS (2 N 64 f32x16 places).
template <int N>
EDF_DEVICE void join_waves(f32x16* x, f32x16* lds, int w, int l) {
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (w >= half && w < 2 * half)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *((f32x4*)(lds) + (((w - half) * N + n) * 4 + r) * 64 + l) =
              f32x4{x[n][4 * r], x[n][4 * r + 1], x[n][4 * r + 2], x[n][4 * r + 3]};
    __syncthreads();
    if (w < half)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 y = *((const f32x4*)(lds) + ((w * N + n) * 4 + r) * 64 + l);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n][4 * r + e] += y[e];
        }
  }
}

// 32 columns (rows of the output) of accumulators X^T [dims][32] to memory, scaled
template <typename T, int HD>
EDF_DEVICE void store_rows_t(T* row, const f32x16* x, float scale, int d, int g) {
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const int c = dt * 32 + 8 * rb + 4 * g;
      if (c < d) {  // d is a multiple of 4
        typedef __attribute__((ext_vector_type(4))) T vec4;
        vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(x[dt][rb * 4 + e] * scale);
        *(vec4*)(row + c) = v;
      }
    }
}

// waves per SIMD that the registers of a kernel leave: operand tensors and accumulators
template <typename T, int HD>
constexpr int waves_per_simd(int tensors, int accumulators) {
  return tensors * HD * (int)sizeof(T) / 256 + accumulators * HD / 64 <= 6 ? 2 : 1;
}

template <typename T, int HD>
__global__ __launch_bounds__(256, (waves_per_simd<T, HD>(3, 1))) void narrow_fwd_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  constexpr bool LDS = sizeof(T) == 2 || HD <= 64;
  using N = NTile<T, HD, LDS>;
  constexpr int TILE = LDS ? N::Tile::ELEMS * (int)sizeof(T) : 0, JOIN = 2 * NDT * 64 * 64;
  __shared__ __attribute__((aligned(16))) char smem[WN_WAVES * TILE > JOIN ? WN_WAVES * TILE : JOIN];
  __shared__ float sM[WN_WAVES][32], sS[WN_WAVES][32];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (a.nx - 1 - xb) * WN_R, myq = q0 + li;
  const T* K = (const T*)a.k + bh / a.G * T_ * d;
  const T* V = (const T*)a.v + bh / a.G * T_ * d;
  T* sv = reinterpret_cast<T*>(smem + w * TILE);

  WFrag<T> qf[NKK], kf[NKK], vf[LDS ? NKK : 1];
  N::rows((const T*)a.q + bh * T_ * d, q0, T_, d, l, qf);
  f32x16 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();
  float m = -INFINITY, lsum = 0.0f;
  const KeyTiles<WN_R, WN_R> kt(q0, T_, a.W, a.S);
  if (w < kt.count) {
    N::rows(K, kt.key0(w), T_, d, l, kf);
    if constexpr (LDS) N::rows(V, kt.key0(w), T_, d, l, vf);
  }
  for (int t = w; t < kt.count; t += WN_WAVES) {
    const int k0 = kt.key0(t);
    const SeesKey sees(myq, k0 + 4 * g, a.W, a.S);
    WFrag<T> vt[LDS ? 1 : 2 * NDT];
    if constexpr (LDS) {
      N::keep(sv, l, vf);
    } else {
#pragma unroll
      for (int j = 0; j < 2 * NDT; ++j) vt[j] = N::trans(V, nullptr, k0, T_, d, j / NDT, j % NDT, l);
    }
    f32x16 s = zero16();
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) s = WFrag<T>::mma(kf[kk], qf[kk], s);
    if (t + WN_WAVES < kt.count) {  // the next tile's loads go out before this one's softmax
      N::rows(K, kt.key0(t + WN_WAVES), T_, d, l, kf);
      if constexpr (LDS) N::rows(V, kt.key0(t + WN_WAVES), T_, d, l, vf);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = sees(d_row(r, 0)) ? s[r] : -INFINITY;
      mx = fmaxf(mx, s[r]);
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
    float rs = 0.0f;  // of P as the product has it: the weights of a row add to one
    WFrag<T> pf[2];
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        rs = pf[kc].set2(e, fast_exp2(fmaf(s[8 * kc + e], a.scale_log2, -mns)),
                         fast_exp2(fmaf(s[8 * kc + e + 1], a.scale_log2, -mns)), rs);
    lsum += rs + __shfl_xor(rs, 32);
    if constexpr (LDS) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int kc = 0; kc < 2; ++kc)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        if constexpr (LDS) o[dt] = WFrag<T>::mma(N::trans(V, sv, k0, T_, d, kc, dt, l), pf[kc], o[dt]);
        else o[dt] = WFrag<T>::mma(vt[kc * NDT + dt], pf[kc], o[dt]);
      }
    if constexpr (LDS) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the waves' maxima, then their sums and outputs in units of the common one
  if (g == 0) sM[w][li] = m;
  __syncthreads();
  const float mm = fmaxf(fmaxf(sM[0][li], sM[1][li]), fmaxf(sM[2][li], sM[3][li]));
  const float f = m == -INFINITY ? 0.0f : fast_exp2((m - mm) * a.scale_log2);
  if (g == 0) sS[w][li] = lsum * f;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] *= f;
  join_waves<NDT>(o, (f32x16*)smem, w, l);
  if (w != 0 || myq >= T_) return;
  const float sum = sS[0][li] + sS[1][li] + sS[2][li] + sS[3][li];
  store_rows_t<T, HD>((T*)a.out + (bh * T_ + myq) * d, o, 1.0f / sum, d, g);
  if (g == 0 && a.lse != nullptr) a.lse[bh * T_ + myq] = (mm * a.scale_log2 + __log2f(sum)) * LN2;
}

template <typename T, int HD>
__global__ __launch_bounds__(256, (waves_per_simd<T, HD>(4, 1))) void narrow_dq_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  using N = NTile<T, HD, true>;
  constexpr int TILE = N::Tile::ELEMS * (int)sizeof(T), JOIN = 2 * NDT * 64 * 64;
  __shared__ __attribute__((aligned(16))) char smem[WN_WAVES * TILE > JOIN ? WN_WAVES * TILE : JOIN];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (a.nx - 1 - xb) * WN_R, myq = q0 + li;
  const T* K = (const T*)a.k + bh / a.G * T_ * d;
  const T* V = (const T*)a.v + bh / a.G * T_ * d;
  T* sk = reinterpret_cast<T*>(smem + w * TILE);

  WFrag<T> qf[NKK], of[NKK], kf[NKK], vf[NKK];
  N::rows((const T*)a.q + bh * T_ * d, q0, T_, d, l, qf);
  N::rows((const T*)a.go + bh * T_ * d, q0, T_, d, l, of);
  N::rows((const T*)a.o + bh * T_ * d, q0, T_, d, l, kf);
  float dd = 0.0f;  // D = dO . O
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
    for (int e = 0; e < 8; ++e) dd = fmaf(kf[kk].get(e), of[kk].get(e), dd);
  dd += __shfl_xor(dd, 32);
  const long qrow = bh * T_ + min(myq, T_ - 1);
  const float lse = a.lse[qrow] * LOG2E;
  if (w == 0 && g == 0 && myq < T_) a.dd[qrow] = dd;
  f32x16 dq[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) dq[dt] = zero16();
  const KeyTiles<WN_R, WN_R> kt(q0, T_, a.W, a.S);
  if (w < kt.count) {
    N::rows(K, kt.key0(w), T_, d, l, kf);
    N::rows(V, kt.key0(w), T_, d, l, vf);
  }
  for (int t = w; t < kt.count; t += WN_WAVES) {
    const int k0 = kt.key0(t);
    const SeesKey sees(myq, k0 + 4 * g, a.W, a.S);
    N::keep(sk, l, kf);
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      s = WFrag<T>::mma(kf[kk], qf[kk], s);
      dp = WFrag<T>::mma(vf[kk], of[kk], dp);
    }
    if (t + WN_WAVES < kt.count) {
      N::rows(K, kt.key0(t + WN_WAVES), T_, d, l, kf);
      N::rows(V, kt.key0(t + WN_WAVES), T_, d, l, vf);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = fast_exp2(fmaf(s[r], a.scale_log2, -lse)) * (dp[r] - dd);  // 1 / sqrt(d) at the end
      s[r] = sees(d_row(r, 0)) ? x : 0.0f;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      WFrag<T> df;
#pragma unroll
      for (int e = 0; e < 8; ++e) df.set(e, s[8 * kc + e]);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) dq[dt] = WFrag<T>::mma(N::trans(K, sk, k0, T_, d, kc, dt, l), df, dq[dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  join_waves<NDT>(dq, (f32x16*)smem, w, l);
  if (w == 0 && myq < T_) store_rows_t<T, HD>((T*)a.dq + qrow * d, dq, a.scale, d, g);
}

// dK, dV parts of 32 sink keys from a chunk of their far queries: the waves divide the chunk's tiles of 32 queries, as
// in the kernels above, with the roles of queries and keys exchanged.  In the dK, dV kernels, whose four waves take 32
// keys of a block each, a few sinks leave three of them idle over all queries (kv_plan has the times of both).  Bound by
// the rows of Q and dO, read a second time: 1x32(8)x8192x128 window 300 37 us, 3.4 TB/s.
template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(256, 1) void window_far_kernel(WindowArgs a) {
  constexpr int NKK = HD / 16, NDT = HD / 32;
  using N = NTile<T, HD, true>;
  constexpr int TILE = N::Tile::ELEMS * (int)sizeof(T), JOIN = 2 * NDT * 64 * 64;
  __shared__ __attribute__((aligned(16))) char smem[2 * WN_WAVES * TILE > JOIN ? 2 * WN_WAVES * TILE : JOIN];
  __shared__ __attribute__((aligned(16))) float sL[WN_WAVES][32], sD[WN_WAVES][32];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;  // batch x key head
  window_block(a, xb, bh);
  const int T_ = a.T, d = a.d;
  const int grp = xb / a.c_far, chunk = xb % a.c_far, key0 = 32 * grp;
  const FarTiles ft(key0 / WINDOW_KB * WINDOW_KB, a.bq, T_, a.W);
  const int t0 = chunk * a.len_far, t1 = min(t0 + a.len_far, ft.n * a.G);
  T* sq = reinterpret_cast<T*>(smem + 2 * w * TILE);
  T* so = reinterpret_cast<T*>(smem + (2 * w + 1) * TILE);

  WFrag<T> kf[NKK], vf[NKK], qf[NKK], of[NKK];
  N::template rows<VEC>((const T*)a.k + bh * T_ * d, key0, T_, d, l, kf);
  N::template rows<VEC>((const T*)a.v + bh * T_ * d, key0, T_, d, l, vf);
  f32x16 dk[NDT], dv[NDT];  // dK^T, dV^T: rows are dims, the column this lane's key
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    dk[dt] = zero16();
    dv[dt] = zero16();
  }
  float rl = 0.0f, rd = 0.0f;
  auto load = [&](int t) {
    const int h = t / ft.n, q0 = ft.qs + (t - h * ft.n) * 32;
    const long base = (bh * a.G + h) * T_;
    N::template rows<VEC>((const T*)a.q + base * d, q0, T_, d, l, qf);
    N::template rows<VEC>((const T*)a.go + base * d, q0, T_, d, l, of);
    const long q = base + min(q0 + li, T_ - 1);
    rl = q0 + li < T_ ? a.lse[q] * LOG2E : INFINITY;  // a query past the end gets P = 0
    rd = a.dd[q];
  };
  if (t0 + w < t1) load(t0 + w);
  for (int t = t0 + w; t < t1; t += WN_WAVES) {
    N::keep(sq, l, qf);
    N::keep(so, l, of);
    if (g == 0) sL[w][li] = rl, sD[w][li] = rd;
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      s = WFrag<T>::mma(qf[kk], kf[kk], s);
      dp = WFrag<T>::mma(of[kk], vf[kk], dp);
    }
    if (t + WN_WAVES < t1) load(t + WN_WAVES);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      const f32x4 lv = *(const f32x4*)(&sL[w][8 * rb + 4 * g]);
      const f32x4 dv4 = *(const f32x4*)(&sD[w][8 * rb + 4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = rb * 4 + e;
        const float p = fast_exp2(fmaf(s[r], a.scale_log2, -lv[e]));
        dp[r] = p * (dp[r] - dv4[e]);  // 1 / sqrt(d) is applied with the sums
        s[r] = p;
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
        dv[dt] = WFrag<T>::mma(N::Tile::trans(so, 16 * kc, dt, l), pf, dv[dt]);
        dk[dt] = WFrag<T>::mma(N::Tile::trans(sq, 16 * kc, dt, l), df, dk[dt]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  join_waves<NDT>(dk, (f32x16*)smem, w, l);
  join_waves<NDT>(dv, (f32x16*)smem, w, l);
  if (w != 0) return;
  const bool sink = key0 + li < a.S;  // the group's other keys are not seen from here
  float* out = a.far + ((bh * a.ng + grp) * a.c_far + chunk) * (64L * HD) + li * HD;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int rb = 0; rb < 4; ++rb) {
      f32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = sink ? dk[dt][rb * 4 + e] : 0.0f;
        y[e] = sink ? dv[dt][rb * 4 + e] : 0.0f;
      }
      *(f32x4*)(out + dt * 32 + 8 * rb + 4 * g) = x;
      *(f32x4*)(out + 32 * HD + dt * 32 + 8 * rb + 4 * g) = y;
    }
}

template <typename T, bool VEC>
void run_far(hipStream_t s, const WindowArgs& a, unsigned grid) {
  switch (window_pad(a.d)) {
    case 32: window_far_kernel<T, 32, VEC><<<grid, 256, 0, s>>>(a); break;
    case 64: window_far_kernel<T, 64, VEC><<<grid, 256, 0, s>>>(a); break;
    case 96: window_far_kernel<T, 96, VEC><<<grid, 256, 0, s>>>(a); break;
    default: window_far_kernel<T, 128, VEC><<<grid, 256, 0, s>>>(a);
  }
}

template <typename T, int HD>
void run(bool backward, hipStream_t s, WindowArgs a, int BH) {
  a.nx = (a.T + WN_R - 1) / WN_R;
  const unsigned grid = (unsigned)a.nx * (unsigned)BH;
  if (backward) narrow_dq_kernel<T, HD><<<grid, 256, 0, s>>>(a);
  else narrow_fwd_kernel<T, HD><<<grid, 256, 0, s>>>(a);
}
template <typename T>
void run_d(bool backward, hipStream_t s, const WindowArgs& a, int BH) {
  switch (window_pad(a.d)) {
    case 32: return run<T, 32>(backward, s, a, BH);
    case 64: return run<T, 64>(backward, s, a, BH);
    case 96: return run<T, 96>(backward, s, a, BH);
    default: return run<T, 128>(backward, s, a, BH);
  }
}

}  // namespace

int window_narrow_run(bool backward, hipStream_t s, const WindowArgs& a, int BH, int dtype) {
  if (dtype == EDF_BF16) run_d<bf16>(backward, s, a, BH);
  else run_d<float>(backward, s, a, BH);
  return check_launch(backward ? "window attention dQ" : "window attention");
}

int window_far_run(hipStream_t s, const WindowArgs& args, int BHkv, int dtype, bool vec) {
  WindowArgs a = args;
  a.nx = a.ng * a.c_far;
  const unsigned grid = (unsigned)a.nx * (unsigned)BHkv;
  if (dtype == EDF_BF16) vec ? run_far<bf16, true>(s, a, grid) : run_far<bf16, false>(s, a, grid);
  else vec ? run_far<float, true>(s, a, grid) : run_far<float, false>(s, a, grid);
  return check_launch("window attention dK, dV of far queries");
}

}  // namespace edf
