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

#include "edf_abi.hpp"
#include "edf_common.hpp"
#include "edf_mfma.hpp"

namespace edf {
namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int PA_WAVES = 4;
constexpr int PA_STEP = 128;                   // chunks are whole steps of four waves' tiles of 32 keys
constexpr int PA_MAX_SPLITS = 255;

struct PagedArgs {
  const void *q, *kc, *vc;
  const int *table, *len;
  void* out;
  float* part;  // [B Hq][splits][d rounded up to 4] outputs, then [B Hq][splits][2] (max in log2 units, sum)
  float* ml;
  int B, Hq, Hkv, G, qt, d, width, block, window, sinks, splits, chunk;
  long num_blocks;
  float scale_log2;
};

// 8 consecutive elements of a row, the K / Q operand of one lane for 32 columns of the contraction
template <typename T> struct Frag;
template <> struct Frag<bf16> {
  bf16x8 v;
  EDF_DEVICE static f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  }
  EDF_DEVICE void set(int e, float x) { v[e] = (bf16)x; }
  EDF_DEVICE void load(const bf16* p) { v = *(const bf16x8*)p; }
  EDF_DEVICE void zero() { v = bf16x8{}; }
  EDF_DEVICE void store(bf16* p) const { *(bf16x8*)p = v; }
};
template <> struct Frag<float> {
  f32x4 lo, hi;
  EDF_DEVICE static f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], c, 0, 0, 0);
    return c;
  }
  EDF_DEVICE void set(int e, float x) {
    if (e < 4) lo[e] = x;
    else hi[e - 4] = x;
  }
  EDF_DEVICE void load(const float* p) {
    lo = *(const f32x4*)p;
    hi = *(const f32x4*)(p + 4);
  }
  EDF_DEVICE void zero() { lo = hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
  EDF_DEVICE void store(float* p) const {
    *(f32x4*)p = lo;
    *(f32x4*)(p + 4) = hi;
  }
};

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

// A wave's tile of 16 NT rows in LDS: row operands, and the transposed operand of 16 dims and keys 4 g .. + 3 of each
// 16, with P in the same key order.
template <typename T, int HD, int NT>
struct KVTile {
  static constexpr int ROWS = 16 * NT;
  static constexpr int ELEMS = sizeof(T) == 2 ? lds_tile_elems<HD>(ROWS) : ROWS * (HD + 4);
  EDF_DEVICE static int off(int row, int col) {
    if constexpr (sizeof(T) == 2) return lds_off<HD>(row, col);
    else return row * (HD + 4) + col;
  }
  EDF_DEVICE static Frag<T> row(const T* t, int r, int col) {
    Frag<T> f;
    f.load(t + off(r, col));
    return f;
  }
  // o += V^T P^T for dims 16 dt + i; p: the lane's 4 NT probabilities
  EDF_DEVICE static f32x4 pv(const T* t, int dt, int g, int i, const float* p, f32x4 o) {
    if constexpr (sizeof(T) == 2) {
      const int row = 4 * g + (i >> 2), col = 16 * dt + 4 * (i & 3);
      if constexpr (NT == 2) {
        Frag<T> v, hi, lo;
        v.v = cat4(lds_read_tr16(t + off(row, col)), lds_read_tr16(t + off(row + 16, col)));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          hi.set(e, p[e]);
          lo.set(e, p[e] - (float)hi.v[e]);
        }
        return Frag<T>::mma(v, hi, Frag<T>::mma(v, lo, o));
      } else {
        typedef __attribute__((ext_vector_type(4))) short s16x4;
        const s16x4 v = __builtin_bit_cast(s16x4, lds_read_tr16(t + off(row, col)));
        bf16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          hi[e] = (bf16)p[e];
          lo[e] = (bf16)(p[e] - (float)hi[e]);
        }
        o = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(s16x4, lo), o, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, __builtin_bit_cast(s16x4, hi), o, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o = __builtin_amdgcn_mfma_f32_16x16x4f32(t[off(16 * n + 4 * g + e, 16 * dt + i)], p[4 * n + e], o, 0, 0, 0);
      return o;
    }
  }
};

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

  // join the four waves: O^T as [query][dim] rows of HD + 4 floats, then each thread sums its elements
  float* so = reinterpret_cast<float*>(smem + w * WAVE_BYTES);
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(so + i * (HD + 4) + 16 * dt + 4 * g) = o[dt];
  if (g == 0) {
    sML[w][i][0] = m == -INFINITY ? -INFINITY : m * a.scale_log2;
    sML[w][i][1] = lsum;
  }
  __syncthreads();
  for (int e = tid; e < nq * a.d; e += 256) {
    const int q = e / a.d, c = e - q * a.d;
    float mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < PA_WAVES; ++x) mm = fmaxf(mm, sML[x][q][0]);
    float acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < PA_WAVES; ++x) {
      const float f = mm == -INFINITY ? 0.0f : fast_exp2(sML[x][q][0] - mm);
      sum = fmaf(f, sML[x][q][1], sum);
      acc = fmaf(f, reinterpret_cast<const float*>(smem + x * WAVE_BYTES)[q * (HD + 4) + c], acc);
    }
    const long row = (long)b * a.Hq + hq0 + q;
    if (a.splits == 1) {
      st((T*)a.out, row * a.d + c, sum > 0.0f ? acc / sum : sum == 0.0f ? 0.0f : sum);
    } else {
      const long pr = row * a.splits + split;
      a.part[pr * ((a.d + 3) & ~3) + c] = acc;
      if (c == 0) {
        a.ml[2 * pr] = mm;
        a.ml[2 * pr + 1] = sum;
      }
    }
  }
}

// out[row] = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over the row's chunks: the chunks over PJ_G groups of 32
// lanes, four elements of the head a lane, then the groups in order
constexpr int PJ_G = 8;
template <typename T>
__global__ __launch_bounds__(32 * PJ_G) void paged_join_kernel(PagedArgs a) {
  __shared__ float sw[PA_MAX_SPLITS];
  __shared__ float sr;
  __shared__ f32x4 part[PJ_G][32];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, grp = tid >> 5, c = (blockIdx.y * 32 + (tid & 31)) * 4;
  const float* ml = a.ml + row * a.splits * 2;
  if (tid < 64) {
    float mm = -INFINITY;
    for (int s = tid; s < a.splits; s += 64) mm = fmaxf(mm, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    float sum = 0.0f;
    for (int s = tid; s < a.splits; s += 64) {
      const float f = mm == -INFINITY || ml[2 * s] == -INFINITY ? 0.0f : fast_exp2(ml[2 * s] - mm);
      sw[s] = f;
      sum = fmaf(f, ml[2 * s + 1], sum);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (tid == 0) sr = sum;
  }
  __syncthreads();
  const int dp = (a.d + 3) & ~3;  // row length of the partial outputs
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < a.d) {
    const float* in = a.part + row * a.splits * dp + c;
#pragma unroll 8
    for (int s = grp; s < a.splits; s += PJ_G) acc += sw[s] * *(const f32x4*)(in + (long)s * dp);
  }
  part[grp][tid & 31] = acc;
  __syncthreads();
  if (grp != 0 || c >= a.d) return;
#pragma unroll
  for (int g = 1; g < PJ_G; ++g) acc += part[g][tid];
  const float sum = sr;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < a.d) st((T*)a.out, row * a.d + c + e, sum > 0.0f ? acc[e] / sum : sum == 0.0f ? 0.0f : sum);
}

// Keys per chunk and chunks for the longest request that the table can hold: about PA_WGS workgroups, so that ragged
// requests, whose later chunks are empty, still fill the 512 places of the GPU twice, and chunks of at least PA_MIN
// keys, below which a workgroup's start (length, page, key: three loads that wait for each other) is no longer paid
// for (16x32(8)x128 ragged to 2000: 23.4 us at 256 keys, 20.1 at 512; 8x8(1)x128 to 30000: 22.3 and 21.6; 32x16(2)x256 to
// 4096: 42.2 at 256, 36.7 at 384).
constexpr int PA_WGS = 2560, PA_MIN = 384;
void plan(int B, int Hkv, int qt, long visible, int& chunk, int& splits) {
  const long wgs = (long)B * Hkv * qt;
  const long want = std::max(1L, std::min((long)PA_MAX_SPLITS, (PA_WGS + wgs - 1) / wgs));
  long c = (visible + want - 1) / want;
  // with fewer chunks of PA_MIN keys than CUs, smaller ones, about one a CU (1x8(8)x128 of 600: 11.4 -> 8.5 us), unless one
  // chunk holds them all (no join: 1x32(8)x128 of 200: 7.1 us, 8.7 in two)
  const bool few = visible > PA_MIN && wgs * ((visible + PA_MIN - 1) / PA_MIN) < 256;
  const long least = few ? std::min((long)PA_MIN, (visible * wgs + 255) / 256) : PA_MIN;
  c = std::max(c, least);
  c = (c + PA_STEP - 1) / PA_STEP * PA_STEP;
  chunk = (int)std::min(c, 1L << 30);
  splits = (int)std::max(1L, (visible + chunk - 1) / chunk);
  // An odd number, the last one empty if need be: workgroups go round the eight XCDs in turn, and with four chunks a
  // request all first ones, which are never empty, would fall on two of them (64x32(8)x128 ragged to 4096: 139 us with
  // four chunks, 123 with three).
  if (splits % 2 == 0) ++splits;
}

long visible_keys(long width, int block, int window, int sinks) {
  const long cap = width * block;
  return window > 0 ? std::min(cap, (long)window + sinks) : cap;
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
  // a head count that the call refuses is no plan either (fewer query heads than key heads would divide by none)
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      table_width <= 0 || block_size <= 0 || window < 0 || sinks < 0)
    return 0;
  int chunk, splits;
  edf::plan(batch, num_kv_heads, (num_heads / num_kv_heads + 15) / 16,
            edf::visible_keys(table_width, block_size, window, sinks), chunk, splits);
  return splits == 1 ? 0 : (size_t)batch * num_heads * splits * ((head_dim + 3) / 4 * 4 + 2) * sizeof(float);
}

int edf_paged_attention(void* stream, const void* q, const void* k_cache, const void* v_cache, const int32_t* table,
                        const int32_t* lengths, void* out, void* workspace, size_t workspace_bytes, int batch,
                        int num_heads, int num_kv_heads, int head_dim, long num_blocks, int block_size,
                        int table_width, int window, int sinks, int dtype) {
  using namespace edf;
  EDF_REQUIRE(batch > 0 && num_heads > 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 && block_size > 0 &&
                  table_width > 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(num_heads % num_kv_heads == 0, EDF_ERR_INVALID_ARG, "num_heads %d is no multiple of num_kv_heads %d",
              num_heads, num_kv_heads);
  EDF_REQUIRE(window >= 0 && sinks >= 0, EDF_ERR_INVALID_ARG, "window and sinks must not be negative");
  EDF_REQUIRE(head_dim <= 256, EDF_ERR_UNSUPPORTED, "head_dim %d > 256 unsupported", head_dim);
  EDF_REQUIRE((double)num_blocks * block_size * num_kv_heads < 2147483648.0, EDF_ERR_UNSUPPORTED,
              "the cache has 2^31 or more rows of head_dim");
  EDF_REQUIRE((long)table_width * block_size < (1L << 30), EDF_ERR_UNSUPPORTED,
              "table_width x block_size must be below 2^30");
  EDF_REQUIRE(q && k_cache && v_cache && table && lengths && out, EDF_ERR_INVALID_ARG, "null tensor pointer");
  PagedArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.table = table, a.len = lengths, a.out = out;
  a.B = batch, a.Hq = num_heads, a.Hkv = num_kv_heads, a.G = num_heads / num_kv_heads, a.qt = (a.G + 15) / 16;
  a.d = head_dim, a.width = table_width, a.block = block_size, a.window = window, a.sinks = sinks;
  a.num_blocks = num_blocks;
  a.scale_log2 = LOG2E / sqrtf((float)head_dim);
  plan(batch, num_kv_heads, a.qt, visible_keys(table_width, block_size, window, sinks), a.chunk, a.splits);
  const double wgs = (double)batch * num_kv_heads * a.qt * a.splits;
  EDF_REQUIRE(wgs < 2147483648.0 && (double)batch * num_heads < 2147483648.0, EDF_ERR_UNSUPPORTED,
              "batch x heads too large for one call");
  const size_t need = edf_paged_attention_workspace_bytes(batch, num_heads, num_kv_heads, head_dim, table_width,
                                                          block_size, window, sinks);
  EDF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), EDF_ERR_WORKSPACE,
              "workspace too small: need %zu bytes", need);
  a.part = (float*)workspace;
  a.ml = (float*)workspace + (size_t)batch * num_heads * a.splits * ((head_dim + 3) / 4 * 4);
  const bool vec = (long)head_dim * (dtype == EDF_BF16 ? 2 : 4) % 16 == 0 &&
                   !(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15);
  hipStream_t s = as_stream(stream);
  const unsigned grid = (unsigned)wgs;
  if (dtype == EDF_BF16)
    launch_paged_t<bf16>(s, a, grid, vec);
  else
    launch_paged_t<float>(s, a, grid, vec);
  return check_launch("paged attention");
}

}  // extern "C"
