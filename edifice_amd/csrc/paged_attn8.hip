// Attention of one new token per request over a paged cache of 8-bit numbers (edf_codes.hpp), each page and key head with
// a float32 scale for its keys and one for its values; paged_attn.hip has the formulas and the same over a cache of the
// model's type:
//   s_j = (q . c_j) ks / sqrt(d),  o = sum_j softmax_j(s) vs c'_j,   codes c, c', scales ks, vs of key j's page.
//
// Half the bytes of a bf16 cache, and bound by them.  The codes are exact in bf16, so the matrix products run on bf16
// operands and the scales multiply scores and probabilities, one of each a key: the codes go to bf16 on their way into the
// wave's LDS tiles (half an instruction an element for e4m3, two for whole numbers) and no dequantised value is formed.
// float32 queries and probabilities go through the same products in three bf16 parts each (off by 2^-24), bf16 queries in
// one and probabilities in two (2^-16), so the results' own rounding is the one that shows.
// Tiles, chunks and joins are paged_attn.hip's.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "edf_codes.hpp"
#include "edf_paged.hpp"

namespace edf {
namespace {

// 16 codes of a row from column col on, zeros past d.  VEC: d a multiple of 16 and the cache aligned to 16.
template <int HD, bool VEC>
EDF_DEVICE u32x4 code_piece(const unsigned char* row, int col, int d) {
  if constexpr (VEC) {
    u32x4 c = *(const u32x4*)(row + min(col, d - 16));
    if (d < HD && col >= d) c = u32x4{0, 0, 0, 0};
    return c;
  } else {
    u32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) c[e >> 2] |= (col + e < d ? (unsigned)row[min(col + e, d - 1)] : 0u) << (8 * (e & 3));
    return c;
  }
}

// 8 codes as bf16, exactly
template <int C>
EDF_DEVICE bf16x8 codes_bf16(unsigned lo, unsigned hi) {
  float f[8];
  Codes<C>::unpack4(lo, f);
  Codes<C>::unpack4(hi, f + 4);
  const u32x4 p = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  return __builtin_bit_cast(bf16x8, p);
}

// x as the sum of N bf16 numbers, largest first
template <int N, typename F>
EDF_DEVICE void bf16_parts(float x, F put) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    const bf16 y = (bf16)x;
    put(p, y);
    x -= (float)y;
  }
}

template <typename T, int C, int HD, bool VEC>
__global__ __launch_bounds__(256, 2) void paged_attn8_kernel(PagedArgs a) {
  constexpr int NT = HD > 128 ? 1 : 2, KEYS = 16 * NT, STEP = PA_WAVES * KEYS;
  constexpr int NKK = HD / 32, NDT = HD / 16;
  constexpr int CPR = HD / 16, NV = KEYS * CPR / 64;  // pieces of 16 codes per row, and per lane of a tile
  constexpr int QP = sizeof(T) == 2 ? 1 : 3, PP = sizeof(T) == 2 ? 2 : 3;  // bf16 parts of a query and of P
  using Tile = KVTile<bf16, HD, NT>;
  constexpr int TILE_BYTES = 2 * Tile::ELEMS * 2, OUT_BYTES = 16 * (HD + 4) * 4;
  constexpr int WAVE_BYTES = TILE_BYTES > OUT_BYTES ? TILE_BYTES : OUT_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[PA_WAVES * WAVE_BYTES];
  __shared__ __attribute__((aligned(16))) float sS[PA_WAVES][2][KEYS];
  __shared__ float sML[PA_WAVES][16][2];

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

  Frag<bf16> qf[QP][NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const T* q = (const T*)a.q + ((long)b * a.Hq + hq0 + min(i, nq - 1)) * a.d;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = 32 * kk + 8 * g + e;
      const float x = to_f32(q[min(col, a.d - 1)]);
      bf16_parts<QP>(i < nq && col < a.d ? x : 0.0f, [&](int p, bf16 y) { qf[p][kk].v[e] = y; });
    }
  }
  f32x4 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, lsum = 0.0f;

  // Page and head [num_blocks Hkv] of visible key n, or -1, and its row within the page; one key a lane, repeated every
  // KEYS lanes.
  const int* tb = a.table + (long)b * a.width;
  struct Place {
    int at, off;
  };
  auto place_of = [&](int nbase) {
    const int n = nbase + (l & (KEYS - 1));
    const int key = a.window > 0 ? n + (n >= ns ? skip : 0) : n;
    const int c = key / a.block;
    const int page = tb[min(c, a.width - 1)];
    return Place{n < n1 && page >= 0 && page < a.num_blocks ? page * a.Hkv + h : -1, key - c * a.block};
  };
  const unsigned char *K = (const unsigned char*)a.kc, *V = (const unsigned char*)a.vc;
  u32x4 kr[NV], vr[NV];
  float ksr = 0.0f, vsr = 0.0f;
  auto load_tile = [&](Place p) {  // an absent key reads row 0: it is masked and its value zeroed
    const int rows = p.at < 0 ? 0 : p.at * a.block + p.off;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = l + 64 * n;
      const long r = __shfl(rows, c / CPR);
      kr[n] = code_piece<HD, VEC>(K + r * a.d, c % CPR * 16, a.d);
      vr[n] = code_piece<HD, VEC>(V + r * a.d, c % CPR * 16, a.d);
    }
    ksr = a.ks[max(p.at, 0)];
    vsr = a.vs[max(p.at, 0)];
  };
  bf16* sk = reinterpret_cast<bf16*>(smem + w * WAVE_BYTES);
  bf16* sv = sk + Tile::ELEMS;
  int nb = split * a.chunk + KEYS * w;
  Place here = place_of(nb);
  if (nb < n1) load_tile(here);
  Place next = place_of(nb + STEP);
  for (; nb < n1; nb += STEP) {
    const unsigned long long live = __ballot(here.at >= 0);  // bit k (repeated): key k of the tile
    // absent keys' values and scales as zeros, since a masked P of 0 would keep a NaN
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = l + 64 * n, row = c / CPR, col = c % CPR * 16;
      if (live != ~0ull && !((live >> row) & 1)) vr[n] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        *(bf16x8*)(sk + Tile::off(row, col + 8 * e)) = codes_bf16<C>(kr[n][2 * e], kr[n][2 * e + 1]);
        *(bf16x8*)(sv + Tile::off(row, col + 8 * e)) = codes_bf16<C>(vr[n][2 * e], vr[n][2 * e + 1]);
      }
    }
    if (l < KEYS) {
      sS[w][0][l] = here.at >= 0 ? ksr * a.scale_log2 : 0.0f;
      sS[w][1][l] = here.at >= 0 ? vsr : 0.0f;
    }
    here = next;
    if (nb + STEP < n1) load_tile(here);
    next = place_of(nb + 2 * STEP);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    f32x4 s[NT], vs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const Frag<bf16> kf = Tile::row(sk, 16 * t + i, 32 * kk + 8 * g);
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) s[t] = Frag<bf16>::mma(kf, qf[p][kk], s[t]);
      }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] *= *(const f32x4*)(&sS[w][0][16 * t + 4 * g]);
      vs[t] = *(const f32x4*)(&sS[w][1][16 * t + 4 * g]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (live != ~0ull) s[t][r] = (live >> (16 * t + 4 * g + r)) & 1 ? s[t][r] : -INFINITY;
        mx = fmaxf(mx, s[t][r]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mnew = fmaxf(m, mx);
    const float mns = mnew == -INFINITY ? 0.0f : mnew;
    if (__any(mnew > m)) {
      const float alpha = fast_exp2(m - mns);
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] *= alpha;
    }
    m = mnew;
    float rs = 0.0f;
    bf16 pf[PP][4 * NT];
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
      const float p = fast_exp2(s[e >> 2][e & 3] - mns);
      rs += p;
      bf16_parts<PP>(p * vs[e >> 2][e & 3], [&](int n, bf16 y) { pf[n][e] = y; });
    }
    rs += __shfl_xor(rs, 16);
    lsum += rs + __shfl_xor(rs, 32);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = Tile::template pv_parts<PP>(sv, dt, g, i, pf, o[dt]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  join_waves<T, HD, WAVE_BYTES>(a, smem, sML, o, m, lsum, b, hq0, nq, split);
}

template <typename T, int C, int HD>
void launch_paged8(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec) {
  if (vec) paged_attn8_kernel<T, C, HD, true><<<grid, 256, 0, s>>>(a);
  else paged_attn8_kernel<T, C, HD, false><<<grid, 256, 0, s>>>(a);
}
template <typename T, int C>
void launch_paged8_t(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec) {
  if (a.d <= 64) launch_paged8<T, C, 64>(s, a, grid, vec);
  else if (a.d <= 128) launch_paged8<T, C, 128>(s, a, grid, vec);
  else launch_paged8<T, C, 256>(s, a, grid, vec);
  if (a.splits > 1)
    paged_join_kernel<T><<<dim3((unsigned)(a.B * a.Hq), (unsigned)((a.d + 127) / 128)), 32 * PJ_G, 0, s>>>(a);
}

}  // namespace
}  // namespace edf

extern "C" {

size_t edf_paged_attention8_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim, int table_width,
                                            int block_size, int window, int sinks) {
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
  const int rc = paged_setup(a, q && k_cache && v_cache && k_scale && v_scale && table && lengths && out, workspace,
                             workspace_bytes, batch, num_heads, num_kv_heads, head_dim, num_blocks, block_size,
                             table_width, window, sinks, dtype);
  if (rc) return rc;
  const bool vec = head_dim % 16 == 0 && !(((uintptr_t)k_cache | (uintptr_t)v_cache) & 15);
  const unsigned grid = (unsigned)((long)batch * num_kv_heads * a.qt * a.splits);
  hipStream_t s = as_stream(stream);
  if (dtype == EDF_BF16)
    code == EDF_INT8 ? launch_paged8_t<bf16, EDF_INT8>(s, a, grid, vec) : launch_paged8_t<bf16, EDF_E4M3>(s, a, grid, vec);
  else
    code == EDF_INT8 ? launch_paged8_t<float, EDF_INT8>(s, a, grid, vec) : launch_paged8_t<float, EDF_E4M3>(s, a, grid, vec);
  return check_launch("paged attention, 8 bits");
}

}  // extern "C"
