// Shared by the attention of one token per request over a paged cache, of the model's type or of 8-bit numbers: the
// arguments, the matrix fragments and tiles, the join of waves and of chunks, and how the keys are cut into chunks.
#pragma once

#include <math.h>

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
  const float *ks, *vs;  // scales [num_blocks Hkv] of a cache of 8-bit numbers
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

// The NW waves' results joined: O^T as [query][dim] rows of HD + 4 floats in the wave's part of smem, then each thread
// sums its elements.  m: the running maximum in log2 units; a workgroup that is one of several chunks leaves its sums.
template <typename T, int HD, int WAVE_BYTES, int NW = PA_WAVES>
EDF_DEVICE void join_waves(const PagedArgs& a, char* smem, float (*sML)[16][2], const f32x4* o, float m, float lsum, int b,
                           int hq0, int nq, int split) {
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, g = l >> 4, i = l & 15;
  float* so = reinterpret_cast<float*>(smem + w * WAVE_BYTES);
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt) *(f32x4*)(so + i * (HD + 4) + 16 * dt + 4 * g) = o[dt];
  if (g == 0) {
    sML[w][i][0] = m;
    sML[w][i][1] = lsum;
  }
  __syncthreads();
  for (int e = tid; e < nq * a.d; e += 64 * NW) {
    const int q = e / a.d, c = e - q * a.d;
    float mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) mm = fmaxf(mm, sML[x][q][0]);
    float acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
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

// Bytes of the chunks' sums; 0 where there is one chunk, and for sizes that the call refuses (fewer query heads than key
// heads would divide by none).
size_t paged_workspace(int batch, int num_heads, int num_kv_heads, int head_dim, int table_width, int block_size, int window,
                       int sinks) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || head_dim <= 0 ||
      table_width <= 0 || block_size <= 0 || window < 0 || sinks < 0)
    return 0;
  int chunk, splits;
  plan(batch, num_kv_heads, (num_heads / num_kv_heads + 15) / 16, visible_keys(table_width, block_size, window, sinks),
       chunk, splits);
  return splits == 1 ? 0 : (size_t)batch * num_heads * splits * ((head_dim + 3) / 4 * 4 + 2) * sizeof(float);
}

// The call's checks, and what the kernels take beside the tensors; whole: requests are not cut, whatever their length
int paged_setup(PagedArgs& a, bool whole, bool pointers, void* workspace, size_t workspace_bytes, int batch, int num_heads,
                int num_kv_heads, int head_dim, long num_blocks, int block_size, int table_width, int window, int sinks,
                int dtype) {
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
  EDF_REQUIRE(pointers, EDF_ERR_INVALID_ARG, "null tensor pointer");
  a.B = batch, a.Hq = num_heads, a.Hkv = num_kv_heads, a.G = num_heads / num_kv_heads, a.qt = (a.G + 15) / 16;
  a.d = head_dim, a.width = table_width, a.block = block_size, a.window = window, a.sinks = sinks;
  a.num_blocks = num_blocks;
  a.scale_log2 = LOG2E / sqrtf((float)head_dim);
  plan(batch, num_kv_heads, a.qt, visible_keys(table_width, block_size, window, sinks), a.chunk, a.splits);
  if (whole) a.chunk = 1 << 30, a.splits = 1;
  const double wgs = (double)batch * num_kv_heads * a.qt * a.splits;
  EDF_REQUIRE(wgs < 2147483648.0 && (double)batch * num_heads < 2147483648.0, EDF_ERR_UNSUPPORTED,
              "batch x heads too large for one call");
  const size_t need =
      whole ? 0 : paged_workspace(batch, num_heads, num_kv_heads, head_dim, table_width, block_size, window, sinks);
  EDF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), EDF_ERR_WORKSPACE,
              "workspace too small: need %zu bytes", need);
  a.part = (float*)workspace;
  a.ml = (float*)workspace + (size_t)batch * num_heads * a.splits * ((head_dim + 3) / 4 * 4);
  return EDF_OK;
}

}  // namespace
}  // namespace edf
