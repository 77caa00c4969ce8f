// Shared by the forward and backward of attention with a sliding window and sinks: the arguments, the
// matrix fragments for both element types and the order in which a query block walks its key tiles.
//
// Query i sees key j when j <= i and (i - j < W or j < S).  Query head h reads key head h / G.
#pragma once

#include "edf_abi.hpp"
#include "edf_common.hpp"
#include "edf_mfma.hpp"

namespace edf {

typedef __attribute__((ext_vector_type(4))) float f32x4;

struct WindowArgs {
  const void *q, *k, *v, *o, *go;
  void *out, *dq, *dk, *dv;
  float *lse, *dd;   // [B Hq T]: natural-log row sums; D = rowsum(dO o O) / unscaled
  float* part;       // backward: float32 dK, dV partials of key blocks that several workgroups share
  int T, G, d, W, S;
  int c_sink, c_win, len_sink, len_win, nsb;  // backward: chunks and tiles per chunk of sink / other key blocks
  float scale, scale_log2;
};

constexpr int WINDOW_DMA_T = 1 << 22;  // longest sequence of the DMA kernels: a head's buffer stays below 2^31 bytes

EDF_DEVICE bool window_sees(int q, int key, int W, int S) { return key <= q && (q - key < W || key < S); }
// the same for key first + c of one query, c a constant after unrolling: three values stay in registers
struct SeesKey {
  int rel, out, sink;
  EDF_DEVICE SeesKey(int q, int first, int W, int S) : rel(q - first), out(q - first - W), sink(S - first) {}
  EDF_DEVICE bool operator()(int c) const { return c <= rel && (c > out || c < sink); }
};

// A loop bound in a vector register: branches on it are divergent in the compiler's eyes, which then keeps the
// bodies of a loop apart (as uniform branches they were merged and spilled: 31 registers in the forward at
// head_dim 128, 592 us against 345).
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

}  // namespace edf
