// Attention of one new token per request over a paged key / value cache, with shared key heads and an
// optional window with sinks:
//   o[b, h] = sum_j softmax_j(q[b, h] . k_j / sqrt(d)) v_j,   key head h / G, G = Hq / Hkv query heads each,
// over the keys j < len_b (window W > 0: j >= len_b - W or j < sinks), key j in page table[b][j / block].
// Each key and value is read once for its G query heads: 2 Hkv len d elements a request, 4 G flops per
// element pair (6 G done in bf16), so the kernel is bound by memory up to about G = 40 in bf16.
//
// The visible keys are numbered through (sinks, then the window) and cut into chunks; a workgroup of four
// waves takes one chunk of one key head, each wave tiles of 32 keys (16 where rows are longer than 256 bytes) with an
// online softmax of its own:
//   S^T [16 keys][16 queries] = K Q^T: MFMA 16x16x32, queries padded to 16 columns;
//   O^T [d][16 queries] += V^T P^T: P^T is the S^T registers (a lane holds keys 4 g .. + 3 of each 16),
//   V^T comes by transposed reads in that order.
// Both tiles pass through wave-private LDS: whole rows are read from memory, 16 lanes a row (the matrix operands'
// own pattern, 64-byte pieces of 16 rows, reaches 4.8 TB/s where whole rows reach 5.2), and the loads of the next
// tile go out as soon as this one's registers are in LDS.  Page numbers are looked up one tile further ahead, one key
// per lane, and handed around the wave by shuffles.
// The waves' results are joined in LDS; with more than one chunk the workgroup leaves (O, max, sum) in
// float32 and a second kernel joins the chunks.
// float32 runs the same way on the float32 matrix instructions (eight 16x16x4 per 32 elements).
//
// Scores, softmax and O are float32; in bf16 P goes through the matrix product in two bf16 parts, off by 2^-16 of itself,
// so the result's own rounding is the only one that shows.  One part, 2^-8 off: 64x32(8)x128 ragged to 4096 123.3 us, with
// two 124.1; 3x16(2)x128 to 131000 37.6 and 38.2; 64x64(8)x64 to 4096, whose rows are shortest, 59.5 and 62.0.
// Keys of a page outside [0, num_blocks) are left out, and a request without keys answers with zeros.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "edf_paged.hpp"

namespace edf {
namespace {

// How rows are read: element by element, in 16-byte pieces, or in 16-byte pieces with d = HD (no element past d, and
// the pieces of a row are immediate offsets from one address).
enum { BY_ELEMENT, BY_PIECE, WHOLE };

// columns col .. col + 7 of a row of d elements, zeros past d
template <typename T, int HD, int MODE>
EDF_DEVICE Frag<T> row_frag(const T* row, int col, int d) {
  Frag<T> f;
  if constexpr (MODE == WHOLE) {
    f.load(row + col);
  } else if constexpr (MODE == BY_PIECE && sizeof(T) == 2) {
    f.load(row + min(col, d - 8));
    if (d < HD && col >= d) f.zero();
  } else if constexpr (MODE == BY_PIECE) {
    f.lo = *(const f32x4*)(row + min(col, d - 4));
    f.hi = *(const f32x4*)(row + min(col + 4, d - 4));
    if (d < HD) {
      if (col >= d) f.lo = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (col + 4 >= d) f.hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = to_f32(row[min(col + e, d - 1)]);
      f.set(e, col + e < d ? x : 0.0f);
    }
  }
  return f;
}

template <typename T, int HD, int MODE>
__global__ __launch_bounds__(256, (HD * sizeof(T) > 512 ? 1 : 2)) void paged_attn_kernel(PagedArgs a) {
  constexpr int NT = HD * sizeof(T) > 256 ? 1 : 2, KEYS = 16 * NT, STEP = PA_WAVES * KEYS;
  constexpr int NKK = HD / 32, NDT = HD / 16;
  constexpr int CPR = HD / 8, NV = KEYS * CPR / 64;  // 8-element pieces per row, and per lane of a tile
  using Tile = KVTile<T, HD, NT>;
  constexpr int TILE_BYTES = 2 * Tile::ELEMS * sizeof(T), OUT_BYTES = 16 * (HD + 4) * 4;
  constexpr int WAVE_BYTES = TILE_BYTES > OUT_BYTES ? TILE_BYTES : OUT_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[PA_WAVES * WAVE_BYTES];
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

  const T *Q = (const T*)a.q, *K = (const T*)a.kc, *V = (const T*)a.vc;
  Frag<T> qf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    qf[kk] = row_frag<T, HD, MODE>(Q + ((long)b * a.Hq + hq0 + min(i, nq - 1)) * a.d, 32 * kk + 8 * g, a.d);
    if (i >= nq) qf[kk].zero();
  }
  f32x4 o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, lsum = 0.0f;

  // row of the cache [num_blocks Hkv block] that holds visible key n, or -1; one key a lane, repeated every KEYS
  // lanes.  The table is read before the length is known to cover n (within its width), so that the two loads of a
  // call without a window do not wait for each other.
  const int* tb = a.table + (long)b * a.width;
  auto row_of = [&](int nbase) {
    const int n = nbase + (l & (KEYS - 1));
    const int key = a.window > 0 ? n + (n >= ns ? skip : 0) : n;
    const int c = key / a.block;
    const int page = tb[min(c, a.width - 1)];
    return n < n1 && page >= 0 && page < a.num_blocks ? (page * a.Hkv + h) * a.block + (key - c * a.block) : -1;
  };
  Frag<T> kr[NV], vr[NV];
  auto load_tile = [&](int rows) {  // a row of -1 reads row 0 (masked, or zeroed)
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = l + 64 * n;
      const long r = max(__shfl(rows, c / CPR), 0);
      kr[n] = row_frag<T, HD, MODE>(K + r * a.d, c % CPR * 8, a.d);
      vr[n] = row_frag<T, HD, MODE>(V + r * a.d, c % CPR * 8, a.d);
    }
  };
  T* sk = reinterpret_cast<T*>(smem + w * WAVE_BYTES);
  T* sv = sk + Tile::ELEMS;
  int nb = split * a.chunk + KEYS * w;
  int rows = row_of(nb);
  if (nb < n1) load_tile(rows);
  int rows_next = row_of(nb + STEP);
  for (; nb < n1; nb += STEP) {
    const unsigned long long live = __ballot(rows >= 0);  // bit k (repeated): key k of the tile
    // values of absent keys as zeros, since a masked P of 0 would keep a NaN
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = l + 64 * n, row = c / CPR;
      kr[n].store(sk + Tile::off(row, c % CPR * 8));
      if (live != ~0ull && !((live >> row) & 1)) vr[n].zero();
      vr[n].store(sv + Tile::off(row, c % CPR * 8));
    }
    rows = rows_next;
    if (nb + STEP < n1) load_tile(rows);
    rows_next = row_of(nb + 2 * STEP);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    f32x4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t] = Frag<T>::mma(Tile::row(sk, 16 * t + i, 32 * kk + 8 * g), qf[kk], s[t]);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (live != ~0ull) s[t][r] = (live >> (16 * t + 4 * g + r)) & 1 ? s[t][r] : -INFINITY;
        mx = fmaxf(mx, s[t][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mnew = fmaxf(m, mx);
    const float mns = mnew == -INFINITY ? 0.0f : mnew * a.scale_log2;
    if (__any(mnew > m)) {
      const float alpha = fast_exp2(m * a.scale_log2 - mns);
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] *= alpha;
    }
    m = mnew;
    float p[4 * NT], rs = 0.0f;
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
      p[e] = fast_exp2(fmaf(s[e >> 2][e & 3], a.scale_log2, -mns));
      rs += p[e];
    }
    rs += __shfl_xor(rs, 16);
    lsum += rs + __shfl_xor(rs, 32);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = Tile::pv(sv, dt, g, i, p, o[dt]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  join_waves<T, HD, WAVE_BYTES>(a, smem, sML, o, m == -INFINITY ? -INFINITY : m * a.scale_log2, lsum, b, hq0, nq, split);
}

template <typename T, int HD>
void launch_paged(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec) {
  if (vec && a.d == HD)
    paged_attn_kernel<T, HD, WHOLE><<<grid, 256, 0, s>>>(a);
  else if (vec)
    paged_attn_kernel<T, HD, BY_PIECE><<<grid, 256, 0, s>>>(a);
  else
    paged_attn_kernel<T, HD, BY_ELEMENT><<<grid, 256, 0, s>>>(a);
}
template <typename T>
void launch_paged_t(hipStream_t s, const PagedArgs& a, unsigned grid, bool vec) {
  if (a.d <= 64)
    launch_paged<T, 64>(s, a, grid, vec);
  else if (a.d <= 128)
    launch_paged<T, 128>(s, a, grid, vec);
  else
    launch_paged<T, 256>(s, a, grid, vec);
  if (a.splits > 1)
    paged_join_kernel<T><<<dim3((unsigned)(a.B * a.Hq), (unsigned)((a.d + 127) / 128)), 32 * PJ_G, 0, s>>>(a);
}

}  // namespace
}  // namespace edf

extern "C" {

size_t edf_paged_attention_workspace_bytes(int batch, int num_heads, int num_kv_heads, int head_dim, int table_width,
                                           int block_size, int window, int sinks) {
  return edf::paged_workspace(batch, num_heads, num_kv_heads, head_dim, table_width, block_size, window, sinks);
}

int edf_paged_attention(void* stream, const void* q, const void* k_cache, const void* v_cache, const int32_t* table,
                        const int32_t* lengths, void* out, void* workspace, size_t workspace_bytes, int batch,
                        int num_heads, int num_kv_heads, int head_dim, long num_blocks, int block_size,
                        int table_width, int window, int sinks, int dtype) {
  using namespace edf;
  PagedArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.table = table, a.len = lengths, a.out = out;
  const int rc = paged_setup(a, false, q && k_cache && v_cache && table && lengths && out, workspace, workspace_bytes, batch,
                             num_heads, num_kv_heads, head_dim, num_blocks, block_size, table_width, window, sinks, dtype);
  if (rc) return rc;
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 &&
                   !(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15);
  hipStream_t s = as_stream(stream);
  const unsigned grid = (unsigned)((long)batch * num_kv_heads * a.qt * a.splits);
  if (dtype == EDF_BF16)
    launch_paged_t<bf16>(s, a, grid, vec);
  else
    launch_paged_t<float>(s, a, grid, vec);
  return check_launch("paged attention");
}

}  // extern "C"
