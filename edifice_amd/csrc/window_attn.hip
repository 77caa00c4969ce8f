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
// Scores, softmax and O are float32.  In bf16 P is rounded to bf16 for the product (2^-8 of each term), its
// sum is taken before that.  float32 runs on the float32 matrix instructions.
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
  constexpr int CPR = HD / 8, PIECES = BN * CPR, CPT = (PIECES + 255) / 256;
  using Tile = WTile<T, HD, BN>;
  __shared__ __attribute__((aligned(16))) T sK[2][Tile::ELEMS];
  __shared__ __attribute__((aligned(16))) T sV[2][Tile::ELEMS];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 5, li = l & 31;
  int xb;
  long bh;
  head_block(xb, bh);
  const int T_ = a.T, d = a.d;
  const int q0 = (gridDim.x - 1 - xb) * WA_BM, qw = q0 + 32 * w, myq = qw + li;
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
  WFrag<T> rk[CPT], rv[CPT];
  auto gload = [&](int t) {
    const int k0 = kt.key0(t);
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      const long key = min(k0 + row, T_ - 1);  // rows past the end repeat the last: their scores are masked
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
    const int k0 = kt.key0(t);
    const T *sk = sK[t & 1], *sv = sV[t & 1];
    f32x16 s[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      s[h] = zero16();
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) s[h] = WFrag<T>::mma(Tile::row(sk, h * 32 + li, kk * 16 + 8 * g), qf[kk], s[h]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (MASK) s[h][r] = window_sees(myq, k0 + h * 32 + d_row(r, g), a.W, a.S) ? s[h][r] : -INFINITY;
        mx = fmaxf(mx, s[h][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mnew = fmaxf(m, mx);
    const float mns = mnew == -INFINITY ? 0.0f : mnew * a.scale_log2;
    if (__any(mnew > m)) {  // rescale only when some row maximum grew
      const float alpha = fast_exp2(m * a.scale_log2 - mns);
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    m = mnew;
    float rs = 0.0f;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[h][r] = fast_exp2(fmaf(s[h][r], a.scale_log2, -mns));
        rs += s[h][r];
      }
    lsum += rs + __shfl_xor(rs, 32);
#pragma unroll
    for (int kc = 0; kc < 2 * NH; ++kc) {
      WFrag<T> pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf.set(e, s[kc >> 1][8 * (kc & 1) + e]);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] = WFrag<T>::mma(Tile::trans(sv, 16 * kc, dt, l), pf, o[dt]);
    }
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

template <typename T, int BN, bool VEC>
void launch_fwd(hipStream_t s, const WindowArgs& a, int BH) {
  const dim3 grid((a.T + WA_BM - 1) / WA_BM, BH);
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
  EDF_REQUIRE(head_dim <= 128, EDF_ERR_UNSUPPORTED, "head_dim %d > 128 unsupported", head_dim);
  EDF_REQUIRE(seq_len < (1 << 30), EDF_ERR_UNSUPPORTED, "seq_len must be below 2^30");
  EDF_REQUIRE((long)batch * num_heads <= 65535, EDF_ERR_UNSUPPORTED, "batch x num_heads must be at most 65535");
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
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 && !(ptrs & 15);
  hipStream_t s = as_stream(stream);
  const int BH = batch * num_heads;
  if (dtype == EDF_BF16)
    vec ? launch_fwd<bf16, 64, true>(s, a, BH) : launch_fwd<bf16, 64, false>(s, a, BH);
  else
    vec ? launch_fwd<float, 32, true>(s, a, BH) : launch_fwd<float, 32, false>(s, a, BH);
  return check_launch("window attention");
}

}  // extern "C"
