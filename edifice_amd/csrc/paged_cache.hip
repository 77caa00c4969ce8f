// Paged key / value cache: block tables and slots from request lengths, and the write of new keys and
// values into their pages.  The cache holds pages of `block` tokens, [num_blocks, Hkv, block, d] each for
// keys and values (a head's tokens of one page are contiguous, which is how the attention reads them);
// a request's table row names its pages in order and slot s = page * block + offset names one token.
//
// edf_paged_extend grows request r from old_r to new_r tokens.  Its pages ceil(old / block) ..
// ceil(new / block) - 1 are drawn in request order from the free list, at first_r = sum of the draws of
// the requests before it; token old_r + t gets slot page * block + (position mod block).
// One launch: a workgroup takes 1024 (request, token) pairs, sums the draws of all requests before its
// first (at most a few KB from L2), scans those of its own in LDS, and takes a new page from the free list
// itself, not from the table, so no workgroup waits for another's table entries.  Bound by the launch: at
// 64 requests of 2048 tokens it writes 1 MB.
//
// edf_paged_cache_write moves rows of d elements, 16 bytes a lane where d and the pointers allow; bound by
// memory.
#include <stdint.h>

#include <algorithm>

#include "edf_abi.hpp"
#include "edf_common.hpp"

namespace edf {
namespace {

constexpr int PX_NT = 256;
constexpr int PX_ITEMS = 1024;  // (request, token) pairs per workgroup
constexpr int PW_NT = 256;
constexpr int PW_ITEMS = 4;     // units per thread of the write

struct Pages {
  int have, want;
};
// pages held and wanted by a request, within the table's width
EDF_DEVICE Pages pages_of(int old_len, int new_len, int block, int width) {
  const int o = max(old_len, 0), n = max(new_len, 0);
  Pages p;
  p.have = min(o / block + (o % block != 0), width);
  p.want = max(min(n / block + (n % block != 0), width), p.have);
  return p;
}

EDF_DEVICE int wave_sum_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__global__ __launch_bounds__(PX_NT) void paged_extend_kernel(int* __restrict__ table, const int* __restrict__ old_len,
                                                             const int* __restrict__ new_len,
                                                             const int* __restrict__ free_ids,
                                                             const int* __restrict__ taken, int* __restrict__ slots,
                                                             int* __restrict__ positions, int* __restrict__ used, int R,
                                                             int width, int nfree, int block, int tokens) {
  __shared__ unsigned first[PX_ITEMS];  // list entries gone before each of this workgroup's requests
  __shared__ int wsum[PX_NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const long i0 = (long)blockIdx.x * PX_ITEMS, total = (long)R * tokens;
  const int r0 = (int)(i0 / tokens);
  const int r1 = (int)(min(i0 + PX_ITEMS, total) - 1) / tokens;  // last request
  const int nr = r1 - r0 + 1;
  auto draws = [&](int r) {
    const Pages p = pages_of(old_len[r], new_len[r], block, width);
    return p.want - p.have;
  };
  auto block_sum = [&](int v) {
    v = wave_sum_i(v);
    __syncthreads();
    if (lane == 0) wsum[wv] = v;
    __syncthreads();
    return wsum[0] + wsum[1] + wsum[2] + wsum[3];
  };
  // entries of the list that are gone; entry numbers are unsigned, so that none past 2^31 looks free
  const unsigned start = taken != nullptr ? (unsigned)max(*taken, 0) : 0u;
  int before = 0;
  for (int r = tid; r < r0; r += PX_NT) before += draws(r);
  before = block_sum(before);
  // scan of the workgroup's own requests: PX_ITEMS / PX_NT consecutive ones per thread
  constexpr int PER = PX_ITEMS / PX_NT;
  int mine[PER], run = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int r = tid * PER + e;
    mine[e] = r < nr ? draws(r0 + r) : 0;
    run += mine[e];
  }
  int incl = run;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(incl, o);
    incl += lane >= o ? up : 0;
  }
  __syncthreads();
  if (lane == 63) wsum[wv] = incl;
  __syncthreads();
  unsigned at = start + (unsigned)(before + incl - run);
  for (int w = 0; w < wv; ++w) at += wsum[w];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    first[tid * PER + e] = at;
    at += mine[e];
  }
  __syncthreads();
  if (blockIdx.x == 0) {  // the draws of all requests
    int all = 0;
    for (int r = tid; r < R; r += PX_NT) all += draws(r);
    all = block_sum(all);
    if (tid == 0) *used = (int)min(start + (unsigned)all, (unsigned)INT32_MAX);
  }
#pragma unroll
  for (int e = 0; e < PX_ITEMS / PX_NT; ++e) {
    const long i = i0 + e * PX_NT + tid;
    if (i >= total) break;
    const int r = (int)(i / tokens), t = (int)(i - (long)r * tokens);
    const int o = max(old_len[r], 0), n = max(new_len[r], 0);
    const Pages pg = pages_of(o, n, block, width);
    const unsigned base = first[r - r0];  // free-list entry of page c: base + (c - held)
    auto page_of = [&](int c) {
      if (c < pg.have) return table[(long)r * width + c];
      const unsigned at = base + (unsigned)(c - pg.have);
      return at < (unsigned)nfree ? free_ids[at] : -1;
    };
    const bool there = n > o && t < n - o;
    const int p = there ? o + t : -1;
    int slot = -1;
    if (there) {
      const int c = p / block, off = p - c * block;
      if (c < width) {
        const int page = page_of(c);
        const long s = (long)page * block + off;
        if (page >= 0 && s <= INT32_MAX) slot = (int)s;
        if (off == 0) table[(long)r * width + c] = page;  // the first token of a new page enters it
      }
    }
    slots[i] = slot;
    positions[i] = p;
    if (t == tokens - 1 && n - o > tokens)  // pages past the tokens asked for
      for (int c = (o + tokens - 1) / block + 1; c < pg.want; ++c) table[(long)r * width + c] = page_of(c);
  }
}

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

// U: the type of one unit (16 bytes, or one element)
template <typename U>
__global__ __launch_bounds__(PW_NT) void paged_write_kernel(const U* __restrict__ k, const U* __restrict__ v,
                                                            const int* __restrict__ slots, U* __restrict__ kc,
                                                            U* __restrict__ vc, unsigned total, unsigned units,
                                                            int T, int Hkv, int block, int num_slots) {
  const unsigned i0 = blockIdx.x * (PW_NT * PW_ITEMS) + threadIdx.x;
  U kr[PW_ITEMS], vr[PW_ITEMS];
  long to[PW_ITEMS];
#pragma unroll
  for (int e = 0; e < PW_ITEMS; ++e) {
    const unsigned i = i0 + e * PW_NT;
    to[e] = -1;
    if (i >= total) continue;
    const unsigned row = i / units, u = i - row * units;
    const unsigned bh = row / (unsigned)T, t = row - bh * T;
    const unsigned b = bh / (unsigned)Hkv, h = bh - b * Hkv;
    const int slot = slots[b * T + t];
    if (slot < 0 || slot >= num_slots) continue;
    const int page = slot / block, off = slot - page * block;
    to[e] = (((long)page * Hkv + h) * block + off) * units + u;
    kr[e] = k[i];
    vr[e] = v[i];
  }
#pragma unroll
  for (int e = 0; e < PW_ITEMS; ++e)
    if (to[e] >= 0) {
      kc[to[e]] = kr[e];
      vc[to[e]] = vr[e];
    }
}

}  // namespace
}  // namespace edf

extern "C" {

int edf_paged_extend(void* stream, int32_t* table, const int32_t* old_lengths, const int32_t* new_lengths,
                     const int32_t* free_blocks, const int32_t* taken, int32_t* slots, int32_t* positions,
                     int32_t* used, int requests, int table_width, int num_free, int block_size, int num_tokens) {
  using namespace edf;
  EDF_REQUIRE(requests > 0 && table_width > 0 && block_size > 0 && num_tokens > 0 && num_free >= 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE((long)requests * num_tokens < (1L << 31), EDF_ERR_UNSUPPORTED, "requests x num_tokens must be below 2^31");
  EDF_REQUIRE((long)requests * table_width < (1L << 31), EDF_ERR_UNSUPPORTED,
              "requests x table_width must be below 2^31");
  EDF_REQUIRE(table && old_lengths && new_lengths && (free_blocks || num_free == 0) && slots && positions && used,
              EDF_ERR_INVALID_ARG, "null tensor pointer");
  EDF_REQUIRE(taken != used, EDF_ERR_INVALID_ARG,
              "taken and used must be two places: workgroups read one while the other is written");
  const unsigned grid = (unsigned)(((long)requests * num_tokens + PX_ITEMS - 1) / PX_ITEMS);
  paged_extend_kernel<<<grid, PX_NT, 0, as_stream(stream)>>>(table, old_lengths, new_lengths, free_blocks, taken,
                                                             slots, positions, used, requests, table_width, num_free,
                                                             block_size, num_tokens);
  return check_launch("paged extend");
}

int edf_paged_cache_write(void* stream, const void* k, const void* v, const int32_t* slots, void* k_cache,
                          void* v_cache, long batch, long seq, int num_kv_heads, int head_dim, long num_blocks,
                          int block_size, int dtype) {
  using namespace edf;
  EDF_REQUIRE(batch > 0 && seq > 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 && block_size > 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(k && v && slots && k_cache && v_cache, EDF_ERR_INVALID_ARG, "null tensor pointer");
  EDF_REQUIRE(num_blocks < (1L << 31) && num_blocks * block_size < (1L << 31), EDF_ERR_UNSUPPORTED,
              "num_blocks x block_size must be below 2^31");
  EDF_REQUIRE(batch < (1L << 31) && seq < (1L << 31), EDF_ERR_UNSUPPORTED, "batch and seq must be below 2^31");
  const int es = dtype == EDF_BF16 ? 2 : 4;
  const uintptr_t ptrs = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache;
  const bool vec = (long)head_dim * es % 16 == 0 && !(ptrs & 15);
  const unsigned units = vec ? (unsigned)((long)head_dim * es / 16) : (unsigned)head_dim;
  EDF_REQUIRE((double)batch * seq * num_kv_heads * units < 2147483648.0, EDF_ERR_UNSUPPORTED,
              "k has too many elements for one call");
  const unsigned total = (unsigned)(batch * seq * num_kv_heads * units);
  const unsigned grid = (total + PW_NT * PW_ITEMS - 1) / (PW_NT * PW_ITEMS);
  const int ns = (int)(num_blocks * block_size);
  hipStream_t s = as_stream(stream);
#define EDF_WRITE(U)                                                                                       \
  paged_write_kernel<U><<<grid, PW_NT, 0, s>>>((const U*)k, (const U*)v, slots, (U*)k_cache, (U*)v_cache, total, units, \
                                               (int)seq, num_kv_heads, block_size, ns)
  if (vec)
    EDF_WRITE(u32x4);
  else if (es == 4)
    EDF_WRITE(unsigned);
  else
    EDF_WRITE(unsigned short);
#undef EDF_WRITE
  return check_launch("paged cache write");
}

}  // extern "C"
