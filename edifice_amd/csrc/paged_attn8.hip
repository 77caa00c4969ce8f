// Attention of one new token per request over a paged cache of 8-bit numbers (edf_codes.hpp), each page and key head with
// a float32 scale for its keys and one for its values; paged_attn.hip has the formulas and the same over a cache of the
// model's type:
//   s_j = (q . c_j) ks / sqrt(d),  o = sum_j softmax_j(s) vs c'_j,   codes c, c', scales ks, vs of key j's page.
//
// Half the bytes of a bf16 cache, and bound by them: 64 requests, 32(8)x128, 115000 tokens in pages of 16, int8: 51 us (4.6
// TB/s; a copy reaches 4.89) and 4.0 for the join; 3 requests, 16(2)x128, 237000 tokens in pages of 64, e4m3: 27 (4.4 TB/s)
// and 5.8 for the join of up to 255 chunks.  Float32 queries, which go through the first product in two parts, take 8% more
// (64 requests to 4096 68.6 and 74.0 us a pass).  The codes are exact in float16, so the matrix products run on float16 operands and the scales multiply scores and
// probabilities, one of each a key; no dequantised value is formed.
//   Keys go from memory to the matrix operand: a lane's 16 codes of each 64 of a row are 16 columns of the contraction,
//   and the query has the same order.  A tile's rows are read whole by four lanes each.
//   Values become float16 on their way into the wave's LDS tile, from where transposed reads take them.
// Queries are scaled by a power of two to a largest element of 2^14 .. 2^15, P vs by 2^15 over the query's largest so far (a
// power of two that rises with it and falls as the running maximum leaves it behind), so that float16's range holds them to
// 2^-39 of the largest, whatever the scales of pages that have next to no weight.
// bf16 queries are exact in it; float32 ones, and P vs, go through the products in two parts, off by 2^-23 of themselves.
// Tiles, chunks and joins are paged_attn.hip's, but that fewer requests are cut (whole_requests).
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "edf_codes.hpp"
#include "edf_paged.hpp"

namespace edf {
namespace {

// How rows are read: element by element, in pieces of 16 codes (d a multiple of 16, the cache aligned to 16), or in pieces
// with d = HD (no code past d).
enum { BY_ELEMENT, BY_PIECE, WHOLE };

// 16 codes of a row from column col on, zeros past d
template <int HD, int MODE>
EDF_DEVICE u32x4 code_piece(const unsigned char* row, int col, int d) {
  if constexpr (MODE == WHOLE) {
    return *(const u32x4*)(row + col);
  } else if constexpr (MODE == BY_PIECE) {
    u32x4 c = *(const u32x4*)(row + min(col, d - 16));
    if (col >= d) c = u32x4{0, 0, 0, 0};
    return c;
  } else {
    u32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) c[e >> 2] |= (col + e < d ? (unsigned)row[min(col + e, d - 1)] : 0u) << (8 * (e & 3));
    return c;
  }
}

// x as the sum of N float16 numbers, largest first
template <int N, typename F>
EDF_DEVICE void half_parts(float x, F put) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const _Float16 y = (_Float16)x;
    put(p, y);
    x -= (float)y;
  }
}
// exponent of the least float32 above zero: no P vs is lost to a unit above it
constexpr int LEAST_UNIT = -148;
EDF_DEVICE f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// A wave's values in LDS, float16: a block for each 16 columns, of rows of 48 bytes (16 columns and padding), so that a
// lane's addresses are one base and constants.  16 lanes write 16 bytes each to 16 places of the 64 banks: they hold 64 / HD
// of a row's pieces of each of HD / 64 .. 4 rows, and the blocks' distances are chosen by that.
template <int HD, int KEYS>
struct ValueTile {
  static constexpr int ROW = 24, BLOCK = KEYS * ROW + (HD <= 64 ? 32 : HD <= 128 ? 48 : 8), ELEMS = HD / 16 * BLOCK;
};

// As many workgroups a CU as registers allow: at 128 elements in bf16 a fourth one spills (106 us where three take 70).
template <typename T, int C, int HD, int MODE, int NW>
__global__ __launch_bounds__(
    64 * NW, (NW > PA_WAVES ? 1 : sizeof(T) == 2 && MODE != BY_ELEMENT ? (HD <= 64 ? 4 : HD <= 128 ? 3 : 2) : 2))
void paged_attn8_kernel(PagedArgs a) {
  constexpr int NT = HD > 128 ? 1 : 2, KEYS = 16 * NT, STEP = NW * KEYS;
  constexpr int NKK = HD / 32, NDT = HD / 16;
  constexpr int CPR = HD / 16, NV = KEYS * CPR / 64;  // pieces of 16 codes per row, and per lane of a tile
  constexpr int NK = HD / 64;                         // pieces of a key that a lane reads
  constexpr int QP = sizeof(T) == 2 ? 1 : 2, PP = 2;  // float16 parts of a query and of P vs
  using Tile = ValueTile<HD, KEYS>;
  constexpr int TILE_BYTES = Tile::ELEMS * 2, OUT_BYTES = 16 * (HD + 4) * 4;
  constexpr int WAVE_BYTES = TILE_BYTES > OUT_BYTES ? TILE_BYTES : OUT_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[NW * WAVE_BYTES];
  __shared__ __attribute__((aligned(16))) float sS[NW][2][KEYS];
  __shared__ float sML[NW][16][2];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4, i = l & 15;
  const int split = blockIdx.x % a.splits;
  const int bq = blockIdx.x / a.splits;  // (b, key head, query tile)
  const int qt = bq % a.qt, h = bq / a.qt % a.Hkv, b = bq / a.qt / a.Hkv;
  const int hq0 = h * a.G + 16 * qt, nq = min(16, a.G - 16 * qt);

  const int len = min(max(a.len[b], 0), a.width * a.block);
  const int lo = a.window > 0 ? max(0, len - a.window) : 0;
  const int ns = min(a.sinks, lo);     // sinks outside the window
  const int nvis = ns + (len - lo);    // visible keys; key n is n + (n >= ns ? lo - ns : 0)
  const int skip = lo - ns;
  const int n1 = min((split + 1) * a.chunk, nvis);  // this workgroup's keys: split * chunk .. n1 - 1

  // The contraction takes a key's columns in the order in which a lane reads them: its group's 16 of each 64.
  f16x8 qf[QP][NKK];
  float qscale;  // what a score is multiplied by for the query's power of two
  {
    const T* q = (const T*)a.q + ((long)b * a.Hq + hq0 + min(i, nq - 1)) * a.d;
    float x[NKK][8], top = 0.0f;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      const int col = 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
      if constexpr (MODE == WHOLE) {
        typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T piece;
#pragma unroll
        for (int n = 0; n < (int)sizeof(T) / 2; ++n) {
          const piece p = *(const piece*)(q + col + 4 * n);
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T); ++e) x[kk][4 * n + e] = to_f32(p[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = to_f32(q[min(col + e, a.d - 1)]);
          x[kk][e] = col + e < a.d ? y : 0.0f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[kk][e]));
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e0;
    frexpf(top, &e0);
    const int up = top > 0.0f && top < INFINITY ? 15 - e0 : 0;
    qscale = ldexpf(1.0f, -up);
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        half_parts<QP>(i < nq ? ldexpf(x[kk][e], up) : 0.0f, [&](int p, _Float16 y) { qf[p][kk][e] = y; });
  }
  f32x4 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, lsum = 0.0f;
  int ve = LEAST_UNIT;  // o is in units of 2^(ve - 15): every P vs so far, at the present maximum, is below 2^ve

  // Page and head [num_blocks Hkv] of visible key n, or -1, and its row of the cache; one key a lane, repeated every KEYS
  // lanes.
  const int* tb = a.table + (long)b * a.width;
  struct Place {
    int at, row;
  };
  auto place_of = [&](int nbase) {
    const int n = nbase + (l & (KEYS - 1));
    const int key = a.window > 0 ? n + (n >= ns ? skip : 0) : n;
    const int c = key / a.block;
    const int page = tb[min(c, a.width - 1)];
    const bool there = n < n1 && page >= 0 && page < a.num_blocks;
    const int at = there ? page * a.Hkv + h : -1;
    return Place{at, there ? at * a.block + (key - c * a.block) : 0};
  };
  const unsigned char *K = (const unsigned char*)a.kc, *V = (const unsigned char*)a.vc;
  u32x4 kr[NT][NK], vr[NV];
  float ksr = 0.0f, vsr = 0.0f;
  // an absent key reads row 0: it is masked and its value zeroed
  auto load_k = [&](Place p) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const long r = __shfl(p.row, 16 * t + i);
#pragma unroll
      for (int n = 0; n < NK; ++n) kr[t][n] = code_piece<HD, MODE>(K + r * a.d, 64 * n + 16 * g, a.d);
    }
    ksr = a.ks[max(p.at, 0)];
  };
  auto load_v = [&](Place p) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = l + 64 * n;
      const long r = __shfl(p.row, c / CPR);
      vr[n] = code_piece<HD, MODE>(V + r * a.d, c % CPR * 16, a.d);
    }
    vsr = a.vs[max(p.at, 0)];
  };
  _Float16* sv = reinterpret_cast<_Float16*>(smem + w * WAVE_BYTES);
  _Float16* sput = sv + l % CPR * Tile::BLOCK + l / CPR * Tile::ROW;  // this lane's first piece
  const bf16* sget = (const bf16*)sv + (4 * g + (i >> 2)) * Tile::ROW + 4 * (i & 3);
  int nb = split * a.chunk + KEYS * w;
  Place here = place_of(nb);
  if (nb < n1) {
    load_k(here);
    load_v(here);
  }
  Place next = place_of(nb + STEP);
  for (; nb < n1; nb += STEP) {
    const unsigned live = (unsigned)__ballot(here.at >= 0);  // bit k (repeated): key k of the tile
    const bool more = nb + STEP < n1;
    if (live != ~0u) {  // absent keys' values and scales as zeros, since a masked P of 0 would keep a NaN
      const unsigned mine = live >> (l / CPR);  // from this lane's first row on
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (!(mine & (1u << 64 / CPR * n))) vr[n] = u32x4{0, 0, 0, 0};
      if (here.at < 0) ksr = vsr = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      _Float16* to = sput + 64 / CPR * n * Tile::ROW;
      *(f16x8*)to = Codes<C>::half8(vr[n][0], vr[n][1]);
      *(f16x8*)(to + 8) = Codes<C>::half8(vr[n][2], vr[n][3]);
    }
    if (l < KEYS) {
      sS[w][0][l] = ksr * a.scale_log2;
      sS[w][1][l] = vsr;
    }
    if (more) load_v(next);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 s[NT], vs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f16x8 kf = Codes<C>::half8(kr[t][kk >> 1][2 * (kk & 1)], kr[t][kk >> 1][2 * (kk & 1) + 1]);
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) s[t] = mfma16(kf, qf[p][kk], s[t]);
      }
    if (more) load_k(next);
    here = next;
    next = place_of(nb + 2 * STEP);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] *= *(const f32x4*)(&sS[w][0][16 * t + 4 * g]) * qscale;
      vs[t] = *(const f32x4*)(&sS[w][1][16 * t + 4 * g]);
      if (live != ~0u) {
        const unsigned mine = live >> (4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = mine & (1u << (16 * t + r)) ? s[t][r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[t][r]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mnew = fmaxf(m, mx);
    const float mns = mnew == -INFINITY ? 0.0f : mnew;
    float rs = 0.0f, wx = 0.0f, pv[4 * NT];  // pv: P vs
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
      const float p = fast_exp2(s[e >> 2][e & 3] - mns);
      rs += p;
      pv[e] = p * vs[e >> 2][e & 3];
      wx = fmaxf(wx, pv[e]);
    }
    wx = fmaxf(wx, __shfl_xor(wx, 16));
    wx = fmaxf(wx, __shfl_xor(wx, 32));
    // the unit falls with what the new maximum leaves of the old P vs
    const int kept = ve + (int)ceilf(fmaxf(m - mnew, -1024.0f));
    const int venew = max(max(kept, LEAST_UNIT), wx > 0.0f ? __builtin_amdgcn_frexp_expf(wx) : LEAST_UNIT);
    if (__any(mnew > m || venew > ve)) {
      const float alpha = fast_exp2(m - mns), beta = fast_exp2(m - mns + (float)(ve - venew));
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] *= beta;
    }
    m = mnew;
    ve = venew;
    f16x4 pf[PP][NT];
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e)
      half_parts<PP>(ldexpf(pv[e], 15 - ve), [&](int n, _Float16 y) { pf[n][e >> 2][e & 3] = y; });
    rs += __shfl_xor(rs, 16);
    lsum += rs + __shfl_xor(rs, 32);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const f16x4 v0 = __builtin_bit_cast(f16x4, lds_read_tr16(sget + dt * Tile::BLOCK));
      if constexpr (NT == 2) {
        const f16x4 v1 = __builtin_bit_cast(f16x4, lds_read_tr16(sget + dt * Tile::BLOCK + 16 * Tile::ROW));
        const f16x8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int n = PP - 1; n >= 0; --n)
          o[dt] = mfma16(v, __builtin_shufflevector(pf[n][0], pf[n][1], 0, 1, 2, 3, 4, 5, 6, 7), o[dt]);
      } else {
#pragma unroll
        for (int n = PP - 1; n >= 0; --n) o[dt] = __builtin_amdgcn_mfma_f32_16x16x16f16(v0, pf[n][0], o[dt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) o[dt][r] = ldexpf(o[dt][r], ve - 15);
  join_waves<T, HD, WAVE_BYTES, NW>(a, smem, sML, o, m, lsum, b, hq0, nq, split);
}

// Requests that are not cut: short ones, where the join's launch costs more than chunks save, and longer ones where there
// is a workgroup for each CU without cutting.  A workgroup of eight waves where each has a CU to itself.  In chunks, and
// whole (us a pass, replayed from a graph / one call after the other):
//   1x8(4)x64 of 600 float32 7.9 / 14.4, 7.3 / 10.6;  1x32(8)x128 of 600 8.9 / 14.2, 8.9 / 10.2, of 1270 9.2 / 14.3, 13.3 /
//   12.9;  32x32(8)x128 to 750 15.4, 10.8, to 2040 25.0, 20.6;  64x32(8)x128 to 600 21.5, 14.9 (eight waves 18.0), to 2040
//   35.7, 32.6, to 4096 52.0, 58.1;  256x16(4)x64 to 2040 37.9, 34.8;  40x32(8)x128 to 3100 34.6, 39.7.
constexpr int WHOLE_WAVES = 8, ONE_PER_CU = 256;
bool whole_requests(int batch, int num_heads, int num_kv_heads, int head_dim, int table_width, int block_size, int window,
                    int sinks) {
  if (num_kv_heads <= 0 || num_heads < num_kv_heads || head_dim > 128) return false;
  const long wgs = (long)batch * num_kv_heads * ((num_heads / num_kv_heads + 15) / 16);
  return visible_keys(table_width, block_size, window, sinks) <= (wgs < ONE_PER_CU ? 768 : 2048);
}

template <typename T, int C, int HD, int NW>
void launch_paged8(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec) {
  if (vec && a.d == HD && !((uintptr_t)a.q & 15)) paged_attn8_kernel<T, C, HD, WHOLE, NW><<<grid, 64 * NW, 0, s>>>(a);
  else if (vec) paged_attn8_kernel<T, C, HD, BY_PIECE, NW><<<grid, 64 * NW, 0, s>>>(a);
  else paged_attn8_kernel<T, C, HD, BY_ELEMENT, NW><<<grid, 64 * NW, 0, s>>>(a);
}
template <typename T, int C>
void launch_paged8_t(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec, bool whole) {
  if (whole && grid <= ONE_PER_CU) {
    if (a.d <= 64) launch_paged8<T, C, 64, WHOLE_WAVES>(s, a, grid, vec);
    else launch_paged8<T, C, 128, WHOLE_WAVES>(s, a, grid, vec);
    return;
  }
  if (a.d <= 64) launch_paged8<T, C, 64, PA_WAVES>(s, a, grid, vec);
  else if (a.d <= 128) launch_paged8<T, C, 128, PA_WAVES>(s, a, grid, vec);
  else launch_paged8<T, C, 256, PA_WAVES>(s, a, grid, vec);
  if (a.splits > 1)
    paged_join_kernel<T><<<dim3((unsigned)(a.B * a.Hq), (unsigned)((a.d + 127) / 128)), 32 * PJ_G, 0, s>>>(a);
}

}  // namespace
}  // namespace edf

extern "C" {

size_t edf_paged_attention8_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim, int table_width,
                                            int block_size, int window, int sinks) {
  if (edf::whole_requests(batch, num_heads, num_kv_heads, head_dim, table_width, block_size, window, sinks)) return 0;
  return edf_paged_attention_workspace_bytes(batch, num_heads, num_kv_heads, head_dim, table_width, block_size, window,
                                             sinks);
}

int edf_paged_attention8(void* stream, const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                         const float* v_scale, const int32_t* table, const int32_t* lengths, void* out,
                         void* workspace, size_t workspace_bytes, int batch, int num_heads, int num_kv_heads,
                         int head_dim, long num_blocks, int block_size, int table_width, int window, int sinks,
                         int dtype, int code) {
  using namespace edf;
  EDF_REQUIRE(code == EDF_INT8 || code == EDF_E4M3, EDF_ERR_INVALID_ARG, "code must be 0 (int8) or 1 (e4m3)");
  PagedArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.ks = k_scale, a.vs = v_scale, a.table = table, a.len = lengths, a.out = out;
  const bool whole = whole_requests(batch, num_heads, num_kv_heads, head_dim, table_width, block_size, window, sinks);
  const int rc = paged_setup(a, whole, q && k_cache && v_cache && k_scale && v_scale && table && lengths && out, workspace,
                             workspace_bytes, batch, num_heads, num_kv_heads, head_dim, num_blocks, block_size,
                             table_width, window, sinks, dtype);
  if (rc) return rc;
  const bool vec = head_dim % 16 == 0 && !(((uintptr_t)k_cache | (uintptr_t)v_cache) & 15);
  const unsigned grid = (unsigned)((long)batch * num_kv_heads * a.qt * a.splits);
  hipStream_t s = as_stream(stream);
  if (dtype == EDF_BF16)
    code == EDF_INT8 ? launch_paged8_t<bf16, EDF_INT8>(s, a, grid, vec, whole)
                     : launch_paged8_t<bf16, EDF_E4M3>(s, a, grid, vec, whole);
  else
    code == EDF_INT8 ? launch_paged8_t<float, EDF_INT8>(s, a, grid, vec, whole)
                     : launch_paged8_t<float, EDF_E4M3>(s, a, grid, vec, whole);
  return check_launch("paged attention, 8 bits");
}

}  // extern "C"
