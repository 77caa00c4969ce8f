// Shared by the forward and backward of attention with a sliding window and sinks: the arguments, the
// matrix fragments for both element types and the order in which a query block walks its key tiles.
//
// Query i sees key j when j <= i and (i - j < W or j < S).  Query head h reads key head h / G.
#pragma once

#include <algorithm>

#include "edf_abi.hpp"
#include "edf_common.hpp"
#include "edf_mfma.hpp"

namespace edf {

typedef __attribute__((ext_vector_type(4))) float f32x4;

struct WindowArgs {
  const void *q, *k, *v, *o, *go;
  void *out, *dq, *dk, *dv;
  float *lse, *dd;   // [B Hq T]: natural-log row sums; D = rowsum(dO o O) / unscaled
  float *part, *far;  // backward: float32 dK, dV parts of key blocks, and of sinks from far queries
  int T, G, d, W, S;
  int nx;            // workgroups per head (the grid is one-dimensional: its other axes end at 65535)
  // dK, dV (KvPlan): chunks and tiles per chunk of sink / other key blocks; parts of a head; blocks, 32-key groups,
  // chunks and tiles per chunk of the sinks whose far queries have a kernel of their own; queries of a near tile
  int nsb, c_sink, len_sink, c_win, len_win, slots, fsb, ng, c_far, len_far, bq;
  float scale, scale_log2;
};

constexpr int WINDOW_KB = 128;  // keys of a dK, dV workgroup
// longest sequence of the buffer loads: a head of 512-byte rows below 2^31 bytes
constexpr int WINDOW_VEC_T = (1 << 22) - 1;

EDF_DEVICE bool window_sees(int q, int key, int W, int S) { return key <= q && (q - key < W || key < S); }
// the same for key first + c of one query, c a constant after unrolling: three values stay in registers
struct SeesKey {
  int rel, out, sink;
  EDF_DEVICE SeesKey(int q, int first, int W, int S) : rel(q - first), out(q - first - W), sink(S - first) {}
  EDF_DEVICE bool operator()(int c) const { return c <= rel && (c > out || c < sink); }
};

// The (block, head) of this workgroup: the blocks of a head, and so the heads that share keys, on one XCD.
EDF_DEVICE void window_block(const WindowArgs& a, int& blk, long& head) {
  const int id = remap_xcd(blockIdx.x, gridDim.x);
  blk = id % a.nx;
  head = id / a.nx;
}

// A loop bound in a vector register: branches on it are divergent in the compiler's eyes, which then keeps the
// bodies of a loop apart (as uniform branches they were merged and spilled: 31 registers in the forward at
// head_dim 128, 592 us against 380, both profiled).
EDF_DEVICE int in_vector_register(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// 8 consecutive contraction elements of one row (or column): the operand of one lane for 16 steps of the
// contraction (lane half g holds steps 8 g .. 8 g + 7).  In float32 step pairs {e, 8 + e} go through eight
// 32x32x2 matrix instructions, so both types share one operand layout and one accumulator layout.
template <typename T> struct WFrag;
template <> struct WFrag<bf16> {
  bf16x8 v;
  EDF_DEVICE static f32x16 mma(const WFrag& a, const WFrag& b, f32x16 c) { return mfma32(a.v, b.v, c); }
  EDF_DEVICE void set(int e, float x) { v[e] = (bf16)x; }
  EDF_DEVICE float get(int e) const { return (float)v[e]; }
  EDF_DEVICE void load(const bf16* p) { v = *(const bf16x8*)p; }
  EDF_DEVICE void store(bf16* p) const { *(bf16x8*)p = v; }
  EDF_DEVICE void zero() { v = bf16x8{}; }
  // elements e, e + 1 (e even); returns s plus the sum of the pair as rounded, one dot product.  (Taking the pairs out
  // of the finished vector instead compiles to its first pair four times.)
  EDF_DEVICE float set2(int e, float x, float y, float s) {
    const bf16x2 p = __builtin_bit_cast(bf16x2, pack_bf16x2(x, y));
    v[e] = p[0];
    v[e + 1] = p[1];
    return __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{(bf16)1.0f, (bf16)1.0f}, s, false);
  }
};
template <> struct WFrag<float> {
  f32x4 lo, hi;
  EDF_DEVICE static f32x16 mma(const WFrag& a, const WFrag& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[e], b.lo[e], c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[e], b.hi[e], c, 0, 0, 0);
    return c;
  }
  EDF_DEVICE void set(int e, float x) {
    if (e < 4) lo[e] = x;
    else hi[e - 4] = x;
  }
  EDF_DEVICE float get(int e) const { return e < 4 ? lo[e] : hi[e - 4]; }
  EDF_DEVICE void load(const float* p) {
    lo = *(const f32x4*)p;
    hi = *(const f32x4*)(p + 4);
  }
  EDF_DEVICE void store(float* p) const {
    *(f32x4*)p = lo;
    *(f32x4*)(p + 4) = hi;
  }
  EDF_DEVICE void zero() { lo = hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
  EDF_DEVICE float set2(int e, float x, float y, float s) {
    set(e, x);
    set(e + 1, y);
    return s + (x + y);
  }
};

// N steps use(i, load(i)) with the loads A steps ahead of their use: the barriers keep the compiler from sinking a
// step's LDS reads to its products, whose wait then idles the matrix core (bf16 4x16(4)x2000x96 window 500 backward:
// 260 -> 234 us).  float32 products outlast the reads and gain nothing from more than one step.
template <int N, int A, typename L, typename U>
EDF_DEVICE void ahead(L load, U use) {
  decltype(load(0)) f[A];
#pragma unroll
  for (int i = 0; i < A && i < N; ++i) f[i] = load(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, f[i % A]);
    if (i + A < N) f[i % A] = load(i + A);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename T>
struct Pair {
  WFrag<T> x, y;
};

// Columns col .. col + 7 of a row of d <= HD elements in memory, zeros past d.  VEC: d a multiple of 16
// bytes and the tensor aligned to 16.
template <typename T, int HD, bool VEC>
EDF_DEVICE WFrag<T> window_row(const T* row, int col, int d) {
  WFrag<T> f;
  if constexpr (VEC && sizeof(T) == 2) {
    f.load(row + min(col, d - 8));
    if (d < HD && col >= d) f.zero();
  } else if constexpr (VEC) {
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

// A workgroup of 256 threads moves the R-row tile at row r0 of x [T, d] through registers into an LDS tile of HD columns,
// N pieces of 8 elements a thread; columns past d are zeros, rows past the end zeros or copies of the last (their scores
// are masked).  VEC: buffer loads, whose range check stands in for comparisons on every piece (a head's T d elements
// have to stay below 2^31 bytes).
template <typename T, int HD, int R, bool VEC>
struct TileLoader {
  static constexpr int CPR = HD / 8, PIECES = R * CPR, N = (PIECES + 255) / 256;
  static constexpr bool F32 = sizeof(T) == 4;
  unsigned lo[VEC ? N : 1], hi[VEC && F32 ? N : 1];  // byte offsets of a piece's 16-byte parts from the tile's first row
  int tid, d, T_;
  EDF_DEVICE TileLoader(int tid_, int d_, int t_) : tid(tid_), d(d_), T_(t_) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
        lo[i] = c < PIECES && col < d ? (unsigned)((row * d + col) * (int)sizeof(T)) : OOB_OFF;
        if constexpr (F32) hi[i] = c < PIECES && col + 4 < d ? (unsigned)((row * d + col + 4) * (int)sizeof(T)) : OOB_OFF;
      }
    }
  }
  EDF_DEVICE void load(const T* x, int r0, WFrag<T>* f) const {
    if constexpr (VEC) {
      const rsrc_t rs = make_rsrc(x, (unsigned)T_ * (unsigned)d * (unsigned)sizeof(T));
      const unsigned base = (unsigned)r0 * (unsigned)d * (unsigned)sizeof(T);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(lo[i] + base), 0, 0);
        if constexpr (F32) {
          f[i].lo = __builtin_bit_cast(f32x4, a);
          f[i].hi = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(hi[i] + base), 0, 0));
        } else {
          f[i].v = __builtin_bit_cast(bf16x8, a);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
        if (PIECES % 256 != 0 && c >= PIECES) continue;
        f[i] = window_row<T, HD, false>(x + (long)min(r0 + row, T_ - 1) * d, col, d);
      }
    }
  }
  template <typename Tile>
  EDF_DEVICE void store(T* lds, const WFrag<T>* f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + 256 * i, row = c / CPR, col = c % CPR * 8;
      if (PIECES % 256 != 0 && c >= PIECES) continue;
      f[i].store(lds + Tile::off(row, col));
    }
  }
};

// A row-major LDS tile of R rows: operand reads along rows, and transposed ones (lane column c, the 8 rows
// r0 + 4 g + {0 .. 3} and r0 + 8 + 4 g + {0 .. 3}, the order in which an accumulator's registers hold rows).
template <typename T, int HD, int R>
struct WTile {
  static constexpr int ELEMS = sizeof(T) == 2 ? lds_tile_elems<HD>(R) : R * (HD + 4);
  EDF_DEVICE static int off(int row, int col) {
    if constexpr (sizeof(T) == 2) return lds_off<HD>(row, col);
    else return row * (HD + 4) + col;
  }
  EDF_DEVICE static WFrag<T> row(const T* t, int r, int col) {
    WFrag<T> f;
    f.load(t + off(r, col));
    return f;
  }
  // columns 32 dt + (lane % 32); l: lane
  EDF_DEVICE static WFrag<T> trans(const T* t, int r0, int dt, int l) {
    WFrag<T> f;
    if constexpr (sizeof(T) == 2) {
      const int grp = l >> 4, i16 = l & 15;
      const int r = r0 + 4 * (grp >> 1) + (i16 >> 2), c = dt * 32 + 16 * (grp & 1) + 4 * (i16 & 3);
      f.v = cat4(lds_read_tr16(t + off(r, c)), lds_read_tr16(t + off(r + 8, c)));
    } else {
      const int g = l >> 5, c = dt * 32 + (l & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.lo[e] = t[off(r0 + 4 * g + e, c)];
        f.hi[e] = t[off(r0 + 8 + 4 * g + e, c)];
      }
    }
    return f;
  }
};

// The key tiles (of BN keys) of query block [q0, q0 + BM), in the order they are walked: sinks before the
// window, the window's first tiles and the diagonal ones, of which some (query, key) pairs are hidden, then
// the tiles that every query of the block sees whole.  first_whole: where the latter begin.
template <int BM, int BN>
struct KeyTiles {
  int ns, edge, ne, diag, nd, mid, count, first_whole;
  EDF_DEVICE KeyTiles(int q0, int T, int W, int S) {
    const int end = (min(T, q0 + BM) + BN - 1) / BN;
    const int wt0 = max(0, q0 - W + 1) / BN;            // first tile of the window
    ns = min((min(S, T) + BN - 1) / BN, wt0);
    const int past = q0 + BM - 1 - W;                   // keys up to here are hidden from the last query
    mid = min(max(past < 0 ? 0 : past / BN + 1, wt0), end);
    edge = wt0;
    ne = mid - wt0;
    diag = max(min((q0 + 1) / BN, end), mid);
    nd = end - diag;
    first_whole = ns + ne + nd;
    count = first_whole + diag - mid;
  }
  EDF_DEVICE int key0(int t) const {
    int x = t;
    if (t >= ns) x = edge + t - ns;
    if (t >= ns + ne) x = diag + t - ns - ne;
    if (t >= first_whole) x = mid + t - first_whole;
    return x * BN;
  }
};

// Query tiles of BQ that see a key of block [k0, k0 + KB), n of them per query head, from query k0 on; far: the queries
// past the block's windows, which see its sinks alone, are left out.
template <int KB>
__host__ __device__ inline int query_tiles(int k0, int BQ, int T, int W, int S, bool far) {
  const int end = T - k0;
  return (((k0 < S && !far) || end < KB - 1 + W ? end : KB - 1 + W) + BQ - 1) / BQ;
}

// The key block of workgroup xb of a dK, dV kernel and its share [t0, t1) of the block's (query head, tile) pairs,
// nt tiles a head from query qs on; slot: where its sums go if they are only a part of the block's, else -1.
template <int KB, int BQ>
struct KeyChunk {
  int key0, qs, nt, t0, t1;
  long slot;
  EDF_DEVICE KeyChunk(const WindowArgs& a, int xb, long bh) {
    const bool sink = xb < a.nsb * a.c_sink;
    const int x = sink ? xb : xb - a.nsb * a.c_sink, len = sink ? a.len_sink : a.len_win;
    const int per = sink ? a.c_sink : a.c_win, blk = (sink ? 0 : a.nsb) + x / per;
    key0 = blk * KB;
    qs = key0;
    nt = query_tiles<KB>(key0, BQ, a.T, a.W, a.S, a.ng > 0);
    t0 = x % per * len;
    t1 = min(t0 + len, nt * a.G);
    slot = per > 1 || blk < a.fsb ? bh * a.slots + xb : -1;
  }
};

// The far queries of the sinks of key block k0: from query qs on, n tiles of 32 a head.
struct FarTiles {
  int qs, n;
  EDF_DEVICE FarTiles(int k0, int BQ, int T, int W) {
    qs = k0 + query_tiles<WINDOW_KB>(k0, BQ, T, W, 0, true) * BQ;
    n = max(0, (T - qs + 31) / 32);
  }
};

// dK, dV of the blocks whose sums are in parts: the chunks of the near queries, then those of the far ones, added in
// order, four elements a thread.  A workgroup takes one of the pieces of a block's [dK | dV][key][dim].
template <typename T, int HD, int KB, int BQ>
__global__ __launch_bounds__(256) void window_sum_kernel(WindowArgs a, int blocks) {
  constexpr int PIECES = 2 * KB * HD / 1024;
  const int piece = blockIdx.x % PIECES, kblk = blockIdx.x / PIECES % blocks;
  const long bh = blockIdx.x / PIECES / blocks;  // batch x key head
  const int kb0 = kblk * KB, per = kblk < a.nsb ? a.c_sink : a.c_win, len = kblk < a.nsb ? a.len_sink : a.len_win;
  if (per == 1 && kblk >= a.fsb) return;  // in place already
  const int x0 = kblk < a.nsb ? kblk * a.c_sink : a.nsb * a.c_sink + (kblk - a.nsb) * a.c_win;
  const int tiles = query_tiles<KB>(kb0, BQ, a.T, a.W, a.S, a.ng > 0) * a.G;
  const int n = min(per, (tiles + len - 1) / len);  // chunks that hold a tile
  const int e = (piece * 256 + threadIdx.x) * 4;
  const bool is_v = e >= KB * HD;
  const int key = e / HD % KB, c = e % HD;
  if (kb0 + key >= a.T || c >= a.d) return;
  const float* in = a.part + (bh * a.slots + x0) * (2L * KB * HD) + e;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int i = 0; i < n; ++i) s += *(const f32x4*)(in + i * (2L * KB * HD));
  if (const int grp = (kb0 + key) / 32; grp < a.ng) {
    const int nf = (FarTiles(kb0, BQ, a.T, a.W).n * a.G + a.len_far - 1) / a.len_far;
    const float* far = a.far + (bh * a.ng + grp) * a.c_far * (64L * HD) + (is_v ? 32 * HD : 0) + key % 32 * HD + c;
#pragma unroll 8
    for (int i = 0; i < nf; ++i) s += *(const f32x4*)(far + i * (64L * HD));
  }
  if (!is_v) s *= a.scale;
  T* out = (T*)(is_v ? a.dv : a.dk) + (bh * a.T + kb0 + key) * a.d + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < a.d) out[i] = from_f32<T>(s[i]);
}

struct KvPlan {
  int nkb, nsb, c_sink, c_win, len_sink, len_win;  // key blocks; the chunks of those with sinks and of the others
  int fsb, ng, c_far, len_far;                     // blocks, 32-key groups and chunks of sinks with a kernel of their own
  double rounds, cost;                             // of the GPU's places; in tiles
  int gx() const { return nsb * c_sink + (nkb - nsb) * c_win; }
  // a head's workgroups that may leave parts, and the blocks that may be in parts, from the first
  int slots() const { return (nsb > 0 && c_sink > 1) || (nkb > nsb && c_win > 1) ? gx() : fsb; }
  int blocks() const { return nkb > nsb && c_win > 1 ? nkb : nsb > 0 && c_sink > 1 ? nsb : fsb; }
  size_t part(int KB, int hd) const { return (size_t)slots() * 2 * KB * hd; }
  size_t far(int hd) const { return (size_t)ng * c_far * 64 * hd; }
};
// How many workgroups share the tiles of a block of KB keys.  The GPU runs `slots` workgroups at once, so a call takes
// about ceil(workgroups / slots) rounds of the longest share, and every workgroup of a divided block costs `join`
// tiles more for its float32 sums, written and read again: the division with the least of that is taken.  A sink
// block's tiles are divided into shares no longer than another block's (with many sink keys into longer ones, so
// that there are not more of them than four rounds).
inline KvPlan kv_divide(int heads, int G, int T, int W, int S, int KB, int BQ, int slots, int join) {
  KvPlan best{};
  const int nkb = (T + KB - 1) / KB, nsb = std::min(nkb, (S + KB - 1) / KB);
  const long n_sink = (long)G * ((T + BQ - 1) / BQ);
  const long n_win = std::min(n_sink, (long)G * ((KB - 1 + W + BQ - 1) / BQ));
  for (long c = 1; c <= 64 && c <= n_win; ++c) {
    KvPlan p{nkb, nsb, 1, 1, 0, 0, 0, 0, 0, 0, 0.0, 0.0};
    p.len_win = (int)((n_win + c - 1) / c);
    p.c_win = (int)((n_win + p.len_win - 1) / p.len_win);
    p.len_sink = (int)std::max((long)p.len_win, (n_sink * nsb * heads + 4L * slots - 1) / (4L * slots));
    p.c_sink = (int)std::max(1L, (n_sink + p.len_sink - 1) / p.len_sink);
    const double rounds = std::max(1.0, (double)heads * p.gx() / slots);
    // a last round that is not full counts by half of what it lacks: workgroups end at different times
    const double whole = (double)(long)(rounds + 0.999999);
    p.rounds = rounds;
    p.cost = 0.5 * (rounds + whole) * (std::max(p.len_win, nsb > 0 ? p.len_sink : 0) + 2.0 + (p.c_win > 1 ? join : 0));
    if (c == 1 || p.cost < best.cost) best = p;
  }
  return best;
}
// The far queries of sinks take part in the dK, dV kernel, where 32 keys keep one wave of four busy, or have a kernel
// whose waves divide them (window_far_kernel).  That one costs 12 us of launch and latencies, and reads the queries'
// rows at about 3.6 TB/s.  In the dK, dV kernel their tiles take the time of any others (about 0.9 PFLOP/s in bf16, 0.14
// in float32), and in a call of less than two rounds without them much of the round that they add.  dK and dV together
// with dQ, in the kernel / apart: bf16 1x32(8)x8192x128 window 300 353 / 313 us, 1x16(2)x16384x64 window 2048 650 / 592,
// 4x16(4)x2000x96 window 500 204 / 175, 4x32(8)x4096x128 window 1024 1037 / 1034, 2x16(4)x3000x64 window 700 125 / 143,
// 8x16(4)x1500x64 window 256 129 / 144; float32 1x8(4)x4000x128 window 2000 1122 / 1034, 2x8(4)x1000x64 window 300 96 /
// 107.  Their own kernel has about one workgroup a CU, of at least two tiles a wave (more have more sums to join:
// 4x32(8)x4096x128 54 us, 65 with two a CU), and 64 a group at most, which the sums read one by one.
inline KvPlan kv_plan(int heads, int G, int T, int W, int S, int hd, int KB, int BQ, int es, int slots, int join) {
  const KvPlan with = kv_divide(heads, G, T, W, S, KB, BQ, slots, join);
  const int near = query_tiles<WINDOW_KB>(0, BQ, T, W, 0, true) * BQ;
  if (S == 0 || near >= T) return with;
  KvPlan p = kv_divide(heads, G, T, W, 0, KB, BQ, slots, join);
  const double tile = 8.0 * KB * BQ * hd / (es == 2 ? 0.9e9 : 0.14e9);  // us of the whole GPU
  const double far = (double)heads * G * (T - near);                  // query rows
  const int ng = (S + 31) / 32;
  const double more = far / BQ * with.nsb * tile + (p.rounds < 2.0 ? 0.6 * (with.cost - p.cost) * tile * slots : 0.0);
  if (more < 1.2 * (12.0 + far * ng * 2.0 * hd * es / 3.6e6)) return with;
  p.fsb = with.nsb, p.ng = ng;
  const long n = (long)G * ((T - near + 31) / 32);  // of the first block, which has the most
  const long len = std::max({8L, (long)((double)n * ng * heads / 256.0), (n + 63) / 64});
  p.len_far = (int)((len + 3) / 4 * 4);
  p.c_far = (int)((n + p.len_far - 1) / p.len_far);
  return p;
}

inline int window_pad(int d) { return (d + 31) / 32 * 32; }

// workgroups of a dK, dV kernel that run at once (256 CUs; the registers leave one or two a CU)
template <typename T>
int kv_slots(int hd) {
  return sizeof(T) == 4 && hd > 64 ? 256 : 512;
}
// the cost of a workgroup's sums in tiles of BQ queries: 8 KB HD bytes written and read again against 8 KB BQ HD
// flops, at the rates of a CU (about 40 bytes and 250 float32 or 2000 bf16 flops a cycle)
template <typename T>
int kv_join(int KB, int BQ) {
  return sizeof(T) == 4 ? 2 : 16 * 32 / BQ;
}

// dK, dV sums of the sinks' far queries (window_narrow.hip)
int window_far_run(hipStream_t s, const WindowArgs& a, int BHkv, int dtype, bool vec);

// a dK, dV kernel, the sinks' far queries, and the sums of the blocks that are in parts
template <typename T, int HD, int KB, int BQ, bool VEC, typename F>
int launch_dkdv(hipStream_t s, WindowArgs a, int BHkv, F kernel) {
  const KvPlan p = kv_plan(BHkv, a.G, a.T, a.W, a.S, HD, KB, BQ, sizeof(T), kv_slots<T>(HD), kv_join<T>(KB, BQ));
  a.nsb = p.nsb, a.c_sink = p.c_sink, a.len_sink = p.len_sink, a.c_win = p.c_win, a.len_win = p.len_win;
  a.slots = p.slots(), a.fsb = p.fsb, a.ng = p.ng, a.c_far = p.c_far, a.len_far = p.len_far, a.bq = BQ;
  a.far = a.part + p.part(KB, HD) * BHkv;
  a.nx = p.gx();
  const int blocks = p.blocks();
  const long wgs = (long)a.nx * BHkv, sums = 2L * KB * HD / 1024 * blocks * BHkv, far = (long)p.ng * p.c_far * BHkv;
  EDF_REQUIRE(wgs < (1L << 31) && sums < (1L << 31) && far < (1L << 31), EDF_ERR_UNSUPPORTED,
              "batch x heads x seq_len too large for one call");
  kernel<<<(unsigned)wgs, 256, 0, s>>>(a);
  int rc = check_launch("window attention dK, dV");
  if (!rc && far) rc = window_far_run(s, a, BHkv, sizeof(T) == 2 ? EDF_BF16 : EDF_F32, VEC);
  if (rc || !blocks) return rc;
  window_sum_kernel<T, HD, KB, BQ><<<(unsigned)sums, 256, 0, s>>>(a, blocks);
  return check_launch("window attention dK, dV sums");
}

// The narrow kernels (window_narrow.hip): forward, or dQ with D.  They take the calls whose 128-query workgroups would
// leave the GPU half empty.  Forward, window 256, wide against narrow: 128 wide workgroups bf16 18.8 / 17.5 us
// (1x32x500x128) and 15.4 / 11.5 (x64), float32 64.8 / 45.5 and 37.1 / 25.7; 192 of them bf16 19.7 / 30.5 (1x16x1500x128)
// and 15.8 / 14.6, float32 65.8 / 68.2 and 38.5 / 40.8.
int window_narrow_run(bool backward, hipStream_t s, const WindowArgs& a, int BH, int dtype);
inline bool window_narrow(int BH, int T, bool vec) { return vec && (long)BH * ((T + 127) / 128) < 160; }

}  // namespace edf
