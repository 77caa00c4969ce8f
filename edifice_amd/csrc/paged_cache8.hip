// A paged cache of 8-bit numbers: the write of new keys and values, and reading pages back (of either kind of cache)
// as keys and values of texts laid end to end.
//
// Write.  The tokens of a page and key head share one float32 scale s; a value x is held as rne(x / s) in 8 bits
// (edf_codes.hpp).  The call's tokens of a page need a scale of at least
//   n = max |x| / 127 (whole numbers), or the least power of two from max |x| / 448 on (e4m3: 448 is its largest number,
//   and a power of two costs no precision), never under 2^-100 unless every x is zero.
// A page that the call begins (its first slot is written) takes s = n.  Otherwise s doubles until it is n at least, and
// the codes that the page holds are halved as often and rounded: by doublings alone, so that a code that is rounded
// again and again is never off by more than one step (1/2 + 1/4 + ...), and e4m3 codes lose nothing until they leave its
// range.  A value that is not finite makes the scale NaN, and with it what the page's head stands for.
//
// One group of threads (a wave, or four for pages of many elements) takes the tokens of one page, for keys or values of
// one head: they follow one another in k, [tokens][d], so the group reads them once, finds their largest and, where their
// slots follow one another too, writes the codes from the same registers; to slots in any other order it goes token by
// token.  Where a page's tokens begin is seen from the slots: one whose predecessor's lies in another page.  Bound by memory: 2 or 4 bytes read and one written a value; 8x2048x8x128 in pages of
// 16, three quarters of them real, bf16 to int8 20.1 us, to e4m3 17.5 (3.7 and 4.4 TB/s), float32 to int8 29.5 (4.3): the
// slots, the values and the scale are three loads that wait for one another.
//
// Read.  A workgroup takes 64 rows of the packed texts of one head; each row's page and scales are looked up once (the
// text by binary search over the offsets), then all threads copy.  Bound by memory: 35858 tokens of 8x128 e4m3 to bf16
// 42.6 us (5.2 TB/s), int8 to float32 86 (4.2); a cache of the result's type, bf16 48 and float32 121.
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "edf_abi.hpp"
#include "edf_codes.hpp"

namespace edf {
namespace {

constexpr float LEAST_SCALE = 0x1p-100f;

struct Write8Args {
  const void* x[2];  // keys, values
  void* cache[2];
  float* scale[2];
  const int* slots;
  long T;
  int B, Hkv, d, block, num_slots, seg, nseg;
};

// 8 values from element i on, of which n exist (VEC: all), as they are stored where they are whole pieces
template <typename T, bool VEC>
struct Piece {
  float f[8];
  EDF_DEVICE void load(const T* x, long i, int n) {
    if constexpr (VEC) {
      typedef __attribute__((ext_vector_type(4))) float f32x4;
      const f32x4 lo = *(const f32x4*)(x + i), hi = *(const f32x4*)(x + i + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = lo[e], f[e + 4] = hi[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = e < n ? to_f32(x[i + e]) : 0.0f;
    }
  }
  EDF_DEVICE float get(int e) const { return f[e]; }
};
template <>
struct Piece<bf16, true> {
  bf16x8 v;
  EDF_DEVICE void load(const bf16* x, long i, int) { v = *(const bf16x8*)(x + i); }
  EDF_DEVICE float get(int e) const { return (float)v[e]; }
};

// the scale that values up to amax need
template <int C>
EDF_DEVICE float least_scale(float amax) {
  if (!(amax < INFINITY)) return __builtin_nanf("");
  if (amax == 0.0f) return 0.0f;
  if constexpr (C == EDF_INT8) return fmaxf(amax * (1.0f / 127.0f), LEAST_SCALE);
  int e;
  const float m = frexpf(amax, &e);  // amax = m 2^e with m in [1/2, 1); 448 = 7/8 2^9
  return ldexpf(1.0f, max(e - 9 + (m > 0.875f), -100));
}

// G threads a run (64: the waves of a workgroup take a run each), which keep REG pieces of 8 values each between the maximum
// and the codes and read what is more again; VEC: d a multiple of 8 and everything aligned to 16.  Four workgroups a CU: six
// are no faster, and eight spill.
template <typename T, int C, int G, int REG, bool VEC>
__global__ __launch_bounds__(256, 4) void paged_write8_kernel(Write8Args a) {
  __shared__ float smax[4];
  const int lane = threadIdx.x & 63, tid = G == 64 ? lane : threadIdx.x;
  const long unit = G == 64 ? (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
  const int which = (int)(unit & 1);
  const long rest = unit >> 1, bh = rest / a.nseg;
  const int h = (int)(bh % a.Hkv);
  const long b = bh / a.Hkv, t0 = rest % a.nseg * a.seg;
  if (b >= a.B) return;  // the last workgroup's waves past the end (G == 64 alone: no barrier follows there)
  const int* slots = a.slots + b * a.T;
  auto slot_at = [&](long t) {
    const int s = t >= 0 && t < a.T ? slots[t] : -1;
    return s >= 0 && s < a.num_slots ? s : -1;
  };
  const int mine = slot_at(t0 + lane), before = slot_at(t0 + lane - 1);
  const int mine0 = max(mine, 0) / a.block * a.block;  // the first slot of this lane's page (-1 lies in none)
  unsigned long long starts =
      __ballot(lane < a.seg && mine >= 0 && !(before >= 0 && (unsigned)(before - mine0) < (unsigned)a.block));
  float* scales = a.scale[which];
  unsigned char* cache = (unsigned char*)a.cache[which];
  while (starts) {
    const int e = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int slot0 = __builtin_amdgcn_readlane(mine, e), first = __builtin_amdgcn_readlane(mine0, e), page = first / a.block, off = slot0 - first;
    // the run: tokens whose slots lie in the page
    int n = 0;
    bool follow = true, fresh = false;  // the slots follow one another; the page's first one is among them
    for (int base = 0;; base += 64) {   // lanes hold the slots of tokens t0 + base + lane
      const int v = base == 0 ? mine : slot_at(t0 + base + lane), pos = e + n - base;
      const unsigned long long ends = ~(__ballot(v >= 0 && (unsigned)(v - first) < (unsigned)a.block) >> pos);
      const int ones = ends ? __builtin_ctzll(ends) : 64;
      const unsigned long long run = ones < 64 ? (1ull << ones) - 1 : ~0ull;
      follow &= (~(__ballot((unsigned)v == (unsigned)slot0 + base + lane - e) >> pos) & run) == 0;
      fresh |= (__ballot(v == first) >> pos & run) != 0;
      n += ones;
      if (ones < 64 - pos || n >= a.block) break;
    }
    n = min(n, a.block);
    const int count = n * a.d;
    const T* x = (const T*)a.x[which] + (bh * a.T + t0 + e) * a.d;
    const long place = (long)page * a.Hkv + h;
    const float old = scales[place];
    Piece<T, VEC> keep[REG];
    float amax = 0.0f;
    bool bad = false;
    auto look = [&](const Piece<T, VEC>& f) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        amax = fmaxf(amax, fabsf(f.get(c)));
        bad |= !(fabsf(f.get(c)) < INFINITY);
      }
    };
#pragma unroll
    for (int i = 0; i < REG; ++i) {  // all loads go out before the first is looked at
      const int p = 8 * (tid + G * i);
      keep[i] = Piece<T, VEC>{};
      if (p < count) keep[i].load(x, p, count - p);
    }
#pragma unroll
    for (int i = 0; i < REG; ++i) look(keep[i]);
    for (int p = 8 * (tid + G * REG); p < count; p += 8 * G) {
      Piece<T, VEC> f;
      f.load(x, p, count - p);
      look(f);
    }
    if (bad) amax = INFINITY;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if constexpr (G == 256) {
      __syncthreads();  // the last run's readers are done, and all have read the old scale
      if (lane == 0) smax[threadIdx.x >> 6] = amax;
      __syncthreads();
      amax = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    }
    const float need = least_scale<C>(amax);
    float s = need, shrink = 1.0f;  // what the page's other codes are multiplied by
    if (!fresh && !(old <= 0.0f)) {
      int e0, e1;
      const float m0 = frexpf(old, &e0), m1 = frexpf(need, &e1);
      const int k = need > 0.0f ? max(0, e1 - e0 + (m1 > m0)) : 0;
      s = old + need == old + need ? ldexpf(old, k) : __builtin_nanf("");  // NaN stays
      if (s == s) shrink = ldexpf(1.0f, -k);
    } else if (!fresh) {
      shrink = 0.0f;  // a page of zeros so far
    }
    if (tid == 0) scales[place] = s;
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    unsigned char* codes = cache + place * a.block * a.d;
    const int W = VEC ? 4 : 1, whole = a.block * a.d;
    auto lower = [&](int p) {  // the codes from p on as the page's new scale has them
      unsigned c = 0;
      if (shrink != 0.0f) {
        float f[4];
        Codes<C>::unpack4(VEC ? *(const unsigned*)(codes + p) : codes[p], f);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] *= shrink;
        c = Codes<C>::pack4(f);
      }
      if constexpr (VEC) *(unsigned*)(codes + p) = c;
      else codes[p] = (unsigned char)c;
    };
    if (!follow) {  // the page's codes first, the new ones over them
      if (shrink != 1.0f)
        for (int p = W * tid; p < whole; p += W * G) lower(p);
      __threadfence();
      if constexpr (G == 256) __syncthreads();
      for (int p = W * tid; p < count; p += W * G) {
        const int t = p / a.d, o = slots[t0 + e + t] - first;
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = i < W && inv > 0.0f ? to_f32(x[p + (i < W ? i : 0)]) * inv : 0.0f;
        unsigned char* to = codes + (long)o * a.d + (p - t * a.d);
        const unsigned c = Codes<C>::pack4(y);
        if constexpr (VEC) *(unsigned*)to = c;
        else *to = (unsigned char)c;
      }
      continue;
    }
    auto store = [&](const Piece<T, VEC>& f, int p) {
      float y[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] = inv > 0.0f ? f.get(c) * inv : 0.0f;
      const u32x2 w = {Codes<C>::pack4(y), Codes<C>::pack4(y + 4)};
      unsigned char* to = codes + (long)off * a.d + p;
      if constexpr (VEC) {
        *(u32x2*)to = w;
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (p + c < count) to[c] = (unsigned char)(w[c >> 2] >> (8 * (c & 3)));
      }
    };
#pragma unroll
    for (int i = 0; i < REG; ++i) {
      const int p = 8 * (tid + G * i);
      if (p < count) store(keep[i], p);
    }
    for (int p = 8 * (tid + G * REG); p < count; p += 8 * G) {
      Piece<T, VEC> f;
      f.load(x, p, count - p);
      store(f, p);
    }
    if (shrink != 1.0f)  // the slots of the page that this run does not write
      for (int p = W * tid; p < whole; p += W * G)
        if (p < off * a.d || p >= off * a.d + count) lower(p);
  }
}

template <typename T, int C>
int launch_write8(hipStream_t s, Write8Args a, bool vec) {
  // a wave keeps up to 8 pieces a lane; the runs of pages that hold more take four waves, but for single tokens: few large
  // pages are then not left to few waves (8x2048x8x128 in pages of 128, where there are enough of them: float32 41.4 us, by
  // waves alone 43.1; bf16 33.9 and 33.7)
  const long runs = 2L * a.B * a.Hkv * a.nseg, page = (long)a.block * a.d;
  const bool wide = page > 8L * 64 * 8 && a.T > 1;
  const long grid = wide ? runs : (runs + 3) / 4;
  EDF_REQUIRE(grid < (1L << 31), EDF_ERR_UNSUPPORTED, "k has too many elements for one call");
#define EDF_WRITE8(G, R, V) paged_write8_kernel<T, C, G, R, V><<<(unsigned)grid, 256, 0, s>>>(a)
  if (!vec) {
    if (wide) EDF_WRITE8(256, 8, false);
    else EDF_WRITE8(64, 4, false);
  } else if (wide) {
    EDF_WRITE8(256, 8, true);
  } else if (page > 8L * 64 * 4 && a.T > 1) {
    EDF_WRITE8(64, 8, true);
  } else {
    EDF_WRITE8(64, 4, true);
  }
#undef EDF_WRITE8
  return check_launch("paged cache write, 8 bits");
}

// ---- read ------------------------------------------------------------------------------

constexpr int PR_ROWS = 64;

struct ReadArgs {
  const void *kc, *vc;
  const float *ks, *vs;
  const int *table, *offsets;
  void *k, *v;
  int requests, width, Hkv, d, block;
  long num_blocks, total;
  unsigned nx;  // workgroups a head
};

// C: the code's kind, or -1 for a cache of T itself; pieces of N elements, 16 bytes of the result (VEC), or one
template <typename T, int C, bool VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
  constexpr int N = VEC ? 16 / (int)sizeof(T) : 1;
  __shared__ long src[PR_ROWS];
  __shared__ float sk[PR_ROWS], sv[PR_ROWS];
  const int tid = threadIdx.x, h = blockIdx.x / a.nx;
  const long r0 = (long)(blockIdx.x % a.nx) * PR_ROWS;
  if (tid < PR_ROWS) {
    const long r = r0 + tid;
    int lo = 0, hi = a.requests;  // the last text that begins at r or before it: offsets[lo] <= r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.offsets[mid] <= r) lo = mid;
      else hi = mid;
    }
    const long at = r - a.offsets[lo];
    long from = -1;
    float x = 0.0f, y = 0.0f;
    if (r < a.total && at >= 0 && r < a.offsets[lo + 1] && at < (long)a.width * a.block) {
      const int c = (int)at / a.block, page = a.table[(long)lo * a.width + c];
      if (page >= 0 && page < a.num_blocks) {
        const long place = (long)page * a.Hkv + h;
        from = place * a.block + ((int)at - c * a.block);
        if constexpr (C >= 0) x = a.ks[place], y = a.vs[place];
      }
    }
    src[tid] = from;
    if constexpr (C >= 0) sk[tid] = x, sv[tid] = y;
  }
  __syncthreads();
  const int per = a.d / N, rows = (int)min((long)PR_ROWS, a.total - r0);
  for (int i = tid; i < rows * per; i += 256) {
    const int row = i / per, col = (i - row * per) * N;
    const long from = src[row], to = ((long)h * a.total + r0 + row) * a.d + col;
    const long at = max(from, 0L) * a.d + col;  // a row without a page reads the first one's and writes zeros
    if constexpr (C < 0 && VEC) {
      u32x4 x = *(const u32x4*)((const T*)a.kc + at), y = *(const u32x4*)((const T*)a.vc + at);
      if (from < 0) x = y = u32x4{0, 0, 0, 0};
      *(u32x4*)((T*)a.k + to) = x;
      *(u32x4*)((T*)a.v + to) = y;
    } else if constexpr (C < 0) {
      const T x = ((const T*)a.kc)[at], y = ((const T*)a.vc)[at];
      ((T*)a.k)[to] = from < 0 ? from_f32<T>(0.0f) : x;
      ((T*)a.v)[to] = from < 0 ? from_f32<T>(0.0f) : y;
    } else {
      float f[2][8];
      const unsigned char *kc = (const unsigned char*)a.kc + at, *vc = (const unsigned char*)a.vc + at;
      const u32x2 x = !VEC ? u32x2{*kc, 0} : N == 8 ? *(const u32x2*)kc : u32x2{*(const unsigned*)kc, 0};
      const u32x2 y = !VEC ? u32x2{*vc, 0} : N == 8 ? *(const u32x2*)vc : u32x2{*(const unsigned*)vc, 0};
#pragma unroll
      for (int q = 0; q < (N + 3) / 4; ++q) {
        Codes<C>::unpack4(x[q], f[0] + 4 * q);
        Codes<C>::unpack4(y[q], f[1] + 4 * q);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        T* out = (T*)(w ? a.v : a.k) + to;
        const float s = (w ? sv : sk)[row];
        if constexpr (VEC) {
          typedef __attribute__((ext_vector_type(N))) T piece;
          piece p;
#pragma unroll
          for (int e = 0; e < N; ++e) p[e] = from_f32<T>(from < 0 ? 0.0f : f[w][e] * s);
          *(piece*)out = p;
        } else {
          out[0] = from_f32<T>(from < 0 ? 0.0f : f[w][0] * s);
        }
      }
    }
  }
}

template <typename T>
void launch_read(hipStream_t s, const ReadArgs& a, unsigned grid, int code, bool vec) {
#define EDF_READ(C)                                                       \
  (vec ? paged_read_kernel<T, C, true><<<grid, 256, 0, s>>>(a)            \
       : paged_read_kernel<T, C, false><<<grid, 256, 0, s>>>(a))
  if (code == EDF_INT8) EDF_READ(EDF_INT8);
  else if (code == EDF_E4M3) EDF_READ(EDF_E4M3);
  else EDF_READ(-1);
#undef EDF_READ
}

}  // namespace
}  // namespace edf

extern "C" {

int edf_paged_cache_write8(void* stream, const void* k, const void* v, const int32_t* slots, void* k_cache,
                           void* v_cache, float* k_scale, float* v_scale, long batch, long seq, int num_kv_heads,
                           int head_dim, long num_blocks, int block_size, int dtype, int code) {
  using namespace edf;
  EDF_REQUIRE(batch > 0 && seq > 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 && block_size > 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(code == EDF_INT8 || code == EDF_E4M3, EDF_ERR_INVALID_ARG, "code must be 0 (int8) or 1 (e4m3)");
  EDF_REQUIRE(k && v && slots && k_cache && v_cache && k_scale && v_scale, EDF_ERR_INVALID_ARG, "null tensor pointer");
  EDF_REQUIRE(num_blocks < (1L << 31) && num_blocks * block_size < (1L << 31), EDF_ERR_UNSUPPORTED,
              "num_blocks x block_size must be below 2^31");
  EDF_REQUIRE(batch < (1L << 31) && seq < (1L << 31), EDF_ERR_UNSUPPORTED, "batch and seq must be below 2^31");
  EDF_REQUIRE((long)block_size * head_dim < (1L << 28), EDF_ERR_UNSUPPORTED, "block_size x head_dim must be below 2^28");
  Write8Args a{};
  a.x[0] = k, a.x[1] = v, a.cache[0] = k_cache, a.cache[1] = v_cache, a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.slots = slots, a.T = seq, a.B = (int)batch, a.Hkv = num_kv_heads, a.d = head_dim, a.block = block_size;
  a.num_slots = (int)(num_blocks * block_size);
  a.seg = std::min(block_size, 64);
  EDF_REQUIRE((double)batch * num_kv_heads * ((seq + a.seg - 1) / a.seg) < 1073741824.0, EDF_ERR_UNSUPPORTED,
              "k has too many elements for one call");
  a.nseg = (int)((seq + a.seg - 1) / a.seg);
  const uintptr_t ptrs = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache;
  const bool vec = head_dim % 8 == 0 && !(ptrs & 15);
  hipStream_t s = as_stream(stream);
  if (dtype == EDF_BF16)
    return code == EDF_INT8 ? launch_write8<bf16, EDF_INT8>(s, a, vec) : launch_write8<bf16, EDF_E4M3>(s, a, vec);
  return code == EDF_INT8 ? launch_write8<float, EDF_INT8>(s, a, vec) : launch_write8<float, EDF_E4M3>(s, a, vec);
}

int edf_paged_cache_read(void* stream, const void* k_cache, const void* v_cache, const float* k_scale,
                         const float* v_scale, const int32_t* table, const int32_t* offsets, void* k, void* v,
                         int requests, long total, int num_kv_heads, int head_dim, long num_blocks, int block_size,
                         int table_width, int dtype, int code) {
  using namespace edf;
  EDF_REQUIRE(requests > 0 && total > 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 && block_size > 0 &&
                  table_width > 0,
              EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(code == EDF_INT8 || code == EDF_E4M3 || code == EDF_NO_CODE, EDF_ERR_INVALID_ARG,
              "code must be 0 (int8), 1 (e4m3) or -1 (a cache of dtype)");
  EDF_REQUIRE(k_cache && v_cache && table && offsets && k && v && (code == EDF_NO_CODE || (k_scale && v_scale)),
              EDF_ERR_INVALID_ARG, "null tensor pointer");
  EDF_REQUIRE(num_blocks < (1L << 31) && (double)num_blocks * block_size * num_kv_heads < 9.0e15, EDF_ERR_UNSUPPORTED,
              "num_blocks must be below 2^31");
  EDF_REQUIRE((long)table_width * block_size < (1L << 31), EDF_ERR_UNSUPPORTED,
              "table_width x block_size must be below 2^31");
  EDF_REQUIRE(total < (1L << 31) && head_dim <= (1 << 20), EDF_ERR_UNSUPPORTED, "total must be below 2^31");
  ReadArgs a{};
  a.kc = k_cache, a.vc = v_cache, a.ks = k_scale, a.vs = v_scale, a.table = table, a.offsets = offsets, a.k = k, a.v = v;
  a.requests = requests, a.width = table_width, a.Hkv = num_kv_heads, a.d = head_dim, a.block = block_size;
  a.num_blocks = num_blocks, a.total = total;
  a.nx = (unsigned)((total + PR_ROWS - 1) / PR_ROWS);
  EDF_REQUIRE((double)a.nx * num_kv_heads < 2147483648.0, EDF_ERR_UNSUPPORTED, "total x heads too large for one call");
  const uintptr_t ptrs = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache;
  const int es = dtype == EDF_BF16 ? 2 : 4;
  const bool vec = !(ptrs & 15) && (code == EDF_NO_CODE ? (long)head_dim * es % 16 == 0 : head_dim % 8 == 0);
  const unsigned grid = a.nx * (unsigned)num_kv_heads;
  if (dtype == EDF_BF16) launch_read<bf16>(as_stream(stream), a, grid, code, vec);
  else launch_read<float>(as_stream(stream), a, grid, code, vec);
  return check_launch("paged cache read");
}

}  // extern "C"
