// Head split of an attention projection with the query / key norms and the rotary positions in the
// same pass: x [B, T, (Hq + 2 Hkv) d] -> q [B, Hq, T, d], k, v [B, Hkv, T, d], forward and backward.
//
// For a query or key head row u [d] at position p (v rows are only moved):
//   r = 1 / sqrt(mean(u^2) + eps),  n = u r w            (w [d]; n = u without norms)
//   pair (a, b) of the first rot elements, angle t_i = p f_i:
//   y_a = A (n_a cos t - n_b sin t),  y_b = A (n_b cos t + n_a sin t);  the other elements y = n
// pairs are (i, i + rot / 2) (half layout) or (2 i, 2 i + 1) (interleaved); A scales the rotated part.
// Backward with g = the transposed rotation of dy (scaled by A), xh = u r:
//   du = r (g w - xh mean(g w xh)),  dw = sum over rows of g xh.
//
// Angles: positions are integers and f_i is given in float64, so the whole turns of p f_i / 2 pi are taken
// off in float64 before the float32 sine (a float32 product is off by 0.06 rad at position 10^6).  The
// sines of a token are computed once per workgroup into LDS and serve all its heads.
//
// Bound by memory (forward reads and writes each element once, backward reads x and dy and writes dx).
// A lane owns a unit of two C-element chunks that hold whole pairs (half layout: C elements at i and the C
// at i + rot / 2), so the rotation needs no exchange between lanes and the norm one butterfly over the row's
// lanes; C elements are 16 bytes where widths and pointers allow, else 8 (bf16) or single elements.
#include <stdint.h>

#include <algorithm>

#include "edf_abi.hpp"
#include "edf_common.hpp"

namespace edf {
namespace {

constexpr int RO_NT = 256;
constexpr int RO_BWD_WG = 1024;   // backward workgroups at most (each leaves one partial weight gradient)
constexpr int RO_TABLE = 2048;    // sine table entries (cos, sin) per tile

struct RotaryArgs {
  const char *x, *wq, *wk;
  const double* freq;
  const int* pos;
  char *q, *k, *v, *dx;
  float* part;      // backward: [gridDim.x][2][d] weight-gradient partials (null without norms)
  long tokens;      // B T
  int T, Hq, Hkv, d, rot;
  int tile, units;  // tokens per tile; units per row
  int pos_batch;    // elements between the positions of two batch rows (0: shared)
  float eps, amp;
};

// C elements as they are loaded (16 bytes, 8, or one element) and their float32 values
template <typename T, int C>
struct Chunk {
  typedef __attribute__((ext_vector_type(C))) T vec;
  vec v;
  EDF_DEVICE void ld(const T* p) { v = *reinterpret_cast<const vec*>(p); }
  EDF_DEVICE void get(float* f) const {
#pragma unroll
    for (int i = 0; i < C; ++i) f[i] = (float)v[i];
  }
  static EDF_DEVICE void st(T* p, const float* f) {
    vec u;
#pragma unroll
    for (int i = 0; i < C; ++i) u[i] = (T)f[i];
    *reinterpret_cast<vec*>(p) = u;
  }
};
template <typename T>
struct Chunk<T, 1> {
  T v;
  EDF_DEVICE void ld(const T* p) { v = p[0]; }
  EDF_DEVICE void get(float* f) const { f[0] = to_f32(v); }
  static EDF_DEVICE void st(T* p, const float* f) { p[0] = from_f32<T>(f[0]); }
};

// The two chunks of unit j: element offsets a and b (b < 0: the row ends after a).
template <int C, bool INTER>
EDF_DEVICE void unit_at(int j, int d, int rot, int& a, int& b) {
  if (INTER || 2 * C * j >= rot) {
    a = 2 * C * j;
    b = a + C < d ? a + C : -1;
  } else {
    a = C * j;
    b = rot / 2 + C * j;
  }
}

// rotate the unit's pairs in place: e[0 .. C) is chunk a, e[C .. 2 C) chunk b; cs: the pairs' (cos, sin)
template <int C, bool INTER, bool BACK>
EDF_DEVICE void turn(float* e, const float2* cs) {
#pragma unroll
  for (int p = 0; p < C; ++p) {
    const int ia = INTER ? 2 * p : p, ib = INTER ? 2 * p + 1 : C + p;
    const float c = cs[p].x, s = BACK ? -cs[p].y : cs[p].y;
    const float ya = e[ia] * c - e[ib] * s, yb = e[ib] * c + e[ia] * s;
    e[ia] = ya;
    e[ib] = yb;
  }
}

// sum over the lpr lanes of a row
EDF_DEVICE float row_sum_n(float v, int lpr) {
  for (int o = lpr / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// lpr lanes (a power of two) walk a row, NU units each.  A tile is a.tile tokens with all their heads; a
// thread's first row of a tile is loaded before the tile's sines are computed (more rows ahead cost more in waves per
// SIMD than they hide: 8x2048x(8 + 2 4)x128 bf16 normed backward 57.0 us with four, 51.7 with two, 47.8 with one).
template <typename T, int C, bool INTER, int NU, bool BACK>
__global__ __launch_bounds__(RO_NT, 4) void rotary_kernel(RotaryArgs a, int lpr) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int H = a.Hq + 2 * a.Hkv, npair = a.units * C;
  float2* sCS = reinterpret_cast<float2*>(smem);                           // [tile][npair]
  float* sW = reinterpret_cast<float*>(smem) + 2 * (size_t)a.tile * npair;  // [2][units][2 C], in unit order
  const int tid = threadIdx.x, j0 = tid & (lpr - 1);
  const int step = RO_NT / lpr;  // rows per pass
  const int step_t = step / H, step_h = step % H;
  const T* X = (const T*)a.x;
  const bool norm = a.wq != nullptr;
  const float inv_d = 1.0f / (float)a.d;
  if (norm)
    for (int i = tid; i < 2 * a.units * 2; i += RO_NT) {
      const int which = i / (2 * a.units), c = i % (2 * a.units);
      int oa, ob;
      unit_at<C, INTER>(c >> 1, a.d, a.rot, oa, ob);
      const int o = c & 1 ? ob : oa;
      const T* W = (const T*)(which ? a.wk : a.wq);
#pragma unroll
      for (int e = 0; e < C; ++e)
        sW[(size_t)(which * a.units * 2 + c) * C + e] = o < 0 || o >= a.d ? 0.0f : to_f32(W[o + e]);
    }
  float accq[NU][2 * C] = {}, acck[NU][2 * C] = {};  // BACK: this thread's share of dw
  int ua[NU], ub[NU];                                // its units' chunks; ua < 0: no unit
#pragma unroll
  for (int n = 0; n < NU; ++n) {
    const int j = j0 + lpr * n;
    unit_at<C, INTER>(j, a.d, a.rot, ua[n], ub[n]);
    if (j >= a.units) ua[n] = ub[n] = -1;
  }

  const long ntile = (a.tokens + a.tile - 1) / a.tile;
  for (long tl = blockIdx.x; tl < ntile; tl += gridDim.x) {
    const int tok0 = (int)(tl * a.tile), nt = min(a.tile, (int)a.tokens - tok0);
    const int b0 = tok0 / a.T, p0 = tok0 - b0 * a.T;  // batch row and place of the tile's first token
    int h = (tid / lpr) % H, t = (tid / lpr) / H;
    bool fresh = true;  // the tile's sines are still to be computed
    for (int r0 = 0; r0 < nt * H; r0 += step) {
      Chunk<T, C> u[NU][2], g[NU][2];
      const int tt = t;
      // 0: query head, 1: key, 2: value, -1: past the tile
      const int kind = t >= nt ? -1 : h < a.Hq ? 0 : h < a.Hq + a.Hkv ? 1 : 2;
      int b = b0, place = p0 + t;
      while (place >= a.T) {
        place -= a.T;
        ++b;
      }
      const int hh = h - (kind <= 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hkv);
      const long hrow = (((long)b * (kind <= 0 ? a.Hq : a.Hkv) + hh) * a.T + place) * a.d;
      const long xrow = ((long)(tok0 + t) * H + h) * a.d;
      if (kind >= 0) {
        const T* Y = (const T*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + hrow;
#pragma unroll
        for (int n = 0; n < NU; ++n)
          if (ua[n] >= 0) {
            if (!BACK || (norm && kind < 2)) {
              u[n][0].ld(X + xrow + ua[n]);
              if (ub[n] >= 0) u[n][1].ld(X + xrow + ub[n]);
            }
            if (BACK) {
              g[n][0].ld(Y + ua[n]);
              if (ub[n] >= 0) g[n][1].ld(Y + ub[n]);
            }
          }
      }
      h += step_h;
      t += step_t;
      if (h >= H) h -= H, ++t;
      if (fresh) {
        fresh = false;
        __syncthreads();  // the last tile's sines are read, the weights are written
        for (int i = tid; i < nt * npair; i += RO_NT) {
          const int ti = i / npair, pr = i - ti * npair;
          float2 cs = make_float2(1.0f, 0.0f);
          if (2 * pr < a.rot) {
            int b = b0, place = p0 + ti;
            while (place >= a.T) {
              place -= a.T;
              ++b;
            }
            const int pos = a.pos ? a.pos[(long)b * a.pos_batch + place] : place;
            double turns = (double)pos * (a.freq[pr] * 0.15915494309189535);  // 1 / (2 pi)
            turns -= rint(turns);
            float s, c;
            sincospif(2.0f * (float)turns, &s, &c);
            cs = make_float2(c * a.amp, s * a.amp);
          }
          sCS[i] = cs;
        }
        __syncthreads();
      }
      if (kind < 0) continue;  // the lanes of a row agree
      const bool turned = kind < 2;
      float x[NU][2 * C] = {}, y[NU][2 * C] = {};  // y: BACK, the gradient
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < NU; ++n)
        if (ua[n] >= 0) {
          if (!BACK || (norm && turned)) {
            u[n][0].get(x[n]);
            if (ub[n] >= 0) u[n][1].get(x[n] + C);
          }
          if (BACK) {
            g[n][0].get(y[n]);
            if (ub[n] >= 0) g[n][1].get(y[n] + C);
          }
#pragma unroll
          for (int e = 0; e < 2 * C; ++e) ss = fmaf(x[n][e], x[n][e], ss);
        }
      float r = 1.0f;
      if (norm) r = rsqrtf(row_sum_n(ss, lpr) * inv_d + a.eps);
      float gx = 0.0f;
      if (turned) {
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          if (ua[n] < 0) continue;
          const int j = j0 + lpr * n;
          const float* w = sW + (size_t)(kind * a.units + j) * 2 * C;
          const float2* cs = sCS + tt * npair + j * C;
          if constexpr (!BACK) {
            if (norm)
#pragma unroll
              for (int e = 0; e < 2 * C; ++e) x[n][e] *= r * w[e];
            turn<C, INTER, false>(x[n], cs);
          } else {
            turn<C, INTER, true>(y[n], cs);
            if (norm) {
#pragma unroll
              for (int e = 0; e < 2 * C; ++e) {
                x[n][e] *= r;  // xh
                const float gw = y[n][e] * w[e], dw = y[n][e] * x[n][e];
                accq[n][e] += kind == 0 ? dw : 0.0f;
                acck[n][e] += kind == 1 ? dw : 0.0f;
                gx = fmaf(gw, x[n][e], gx);
                y[n][e] = gw;
              }
            }
          }
        }
        if (BACK && norm) {
          gx = row_sum_n(gx, lpr) * inv_d;
#pragma unroll
          for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int e = 0; e < 2 * C; ++e) y[n][e] = r * fmaf(-x[n][e], gx, y[n][e]);
        }
      }
      T* out = BACK ? (T*)a.dx + xrow : (T*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + hrow;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if (ua[n] < 0) continue;
        const float* f = BACK ? y[n] : x[n];
        Chunk<T, C>::st(out + ua[n], f);
        if (ub[n] >= 0) Chunk<T, C>::st(out + ub[n], f + C);
      }
    }
  }
  if constexpr (BACK) {
    if (a.part == nullptr) return;
    // the workgroup's partial: threads of one unit in row order, through LDS one row group at a time
    float* red = reinterpret_cast<float*>(smem);
    float* out = a.part + (size_t)blockIdx.x * 2 * a.d;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2 * C; ++e) red[e * RO_NT + tid] = which ? acck[n][e] : accq[n][e];
        __syncthreads();
        for (int i = tid; i < lpr * 2 * C; i += RO_NT) {
          const int j = i % lpr, e = i / lpr;
          float s = 0.0f;
          for (int m = 0; m < step; ++m) s += red[e * RO_NT + m * lpr + j];
          const int ju = j + lpr * n;
          if (ju < a.units) {
            int oa, ob;
            unit_at<C, INTER>(ju, a.d, a.rot, oa, ob);
            const int o = e < C ? oa + e : ob < 0 ? -1 : ob + e - C;
            if (o >= 0 && o < a.d) out[which * a.d + o] = s;
          }
        }
      }
  }
}

// dw[c] = sum of the partials in order: one workgroup per 16 columns, 64 partials at a time
template <typename T>
__global__ __launch_bounds__(1024) void rotary_dw_kernel(const float* __restrict__ part, T* dwq, T* dwk, int n, int d) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  float s = 0.0f;
  if (col < 2 * d) {
#pragma unroll 8
    for (int i = r; i < n; i += 64) s += part[(size_t)i * 2 * d + col];
  }
  red[r][c] = s;
  __syncthreads();
  if (r >= 4 || col >= 2 * d) return;
#pragma unroll
  for (int i = 4; i < 64; i += 4) s += red[r + i][c];
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if (r != 0) return;
  if (col < d)
    dwq[col] = from_f32<T>(s);
  else
    dwk[col - d] = from_f32<T>(s);
}

// chunk of C elements: 16 bytes, else 8 (bf16), else one element
int chunk_of(const RotaryArgs& a, bool inter, int es, uintptr_t ptrs) {
  for (int bytes = 16; bytes >= 8; bytes >>= 1) {
    const int c = bytes / es;
    if (es == 4 && c != 4) continue;
    if (a.d % c == 0 && (inter || a.rot / 2 % c == 0) && ptrs % bytes == 0) return c;
  }
  return 1;
}

template <typename T, int C, bool INTER, int NU, bool BACK>
int rotary_launch(hipStream_t s, RotaryArgs a, unsigned max_wg, unsigned* wg) {
  const int half_units = a.rot / (2 * C);
  a.units = INTER ? (a.d + 2 * C - 1) / (2 * C) : half_units + (a.d - a.rot + 2 * C - 1) / (2 * C);
  int lpr = 1;
  while (lpr * NU < a.units) lpr <<= 1;
  const int H = a.Hq + 2 * a.Hkv, npair = a.units * C;
  // Forward: two rows a thread and tile (four: 25.6 us for 24.8 at 8x2048x(8 + 2 4)x128 bf16).  Backward: as many, up to
  // eight, as leave a tile for each of its workgroups, which keep their weight gradients over all their tiles.
  const int step = RO_NT / lpr;
  const int passes = BACK ? (int)std::max(1L, std::min(8L, a.tokens * H / ((long)step * RO_BWD_WG))) : 2;
  int tile = std::max(1, passes * step / H);
  tile = std::min(tile, std::max(1, RO_TABLE / npair));
  a.tile = tile;
  const long ntile = (a.tokens + tile - 1) / tile;
  const unsigned grid = (unsigned)std::min(ntile, (long)max_wg);
  size_t lds = sizeof(float2) * (size_t)tile * npair + (a.wq ? sizeof(float) * 2 * 2 * C * a.units : 0);
  if (BACK && a.part) lds = std::max(lds, sizeof(float) * 2 * C * RO_NT);
  rotary_kernel<T, C, INTER, NU, BACK><<<grid, RO_NT, lds, s>>>(a, lpr);
  *wg = grid;
  return check_launch(BACK ? "rotary head split backward" : "rotary head split");
}

template <bool BACK>
int rotary_dispatch(hipStream_t s, const RotaryArgs& a, bool inter, int dtype, unsigned max_wg, unsigned* wg) {
  const int es = dtype == EDF_BF16 ? 2 : 4;
  uintptr_t ptrs = (uintptr_t)a.x | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.dx;
  const int c = chunk_of(a, inter, es, ptrs);
#define EDF_ROTARY(T, C, NU)                                                        \
  return inter ? rotary_launch<T, C, true, NU, BACK>(s, a, max_wg, wg) : rotary_launch<T, C, false, NU, BACK>(s, a, max_wg, wg)
  if (dtype == EDF_BF16) {
    if (c == 8) EDF_ROTARY(bf16, 8, 1);
    if (c == 4) EDF_ROTARY(bf16, 4, 1);
    EDF_ROTARY(bf16, 1, 2);
  }
  if (c == 4) EDF_ROTARY(float, 4, 1);
  EDF_ROTARY(float, 1, 2);
#undef EDF_ROTARY
}

int rotary_check(const RotaryArgs& a, long B, long T, bool has_wk, int dtype) {
  EDF_REQUIRE(B > 0 && T > 0 && a.Hq > 0 && a.Hkv > 0 && a.d > 0, EDF_ERR_INVALID_ARG, "dimensions must be positive");
  EDF_REQUIRE(valid_dtype(dtype), EDF_ERR_INVALID_ARG, "dtype must be 0 (f32) or 1 (bf16)");
  EDF_REQUIRE(a.d <= 256, EDF_ERR_UNSUPPORTED, "head_dim %d > 256 unsupported", a.d);
  EDF_REQUIRE(a.rot >= 0 && a.rot <= a.d && a.rot % 2 == 0, EDF_ERR_INVALID_ARG,
              "rotary_dim %d must be even and at most head_dim %d", a.rot, a.d);
  EDF_REQUIRE(B < (1L << 31) && T < (1L << 31) && B * T < (1L << 31) && (long)a.Hq + 2L * a.Hkv < (1L << 20),
              EDF_ERR_UNSUPPORTED, "B T must be below 2^31 and the heads below 2^20");
  EDF_REQUIRE(a.x && a.q && a.k && a.v && (a.freq || a.rot == 0), EDF_ERR_INVALID_ARG, "null tensor pointer");
  EDF_REQUIRE((a.wq != nullptr) == has_wk, EDF_ERR_INVALID_ARG, "query and key norm weights come together");
  return EDF_OK;
}

}  // namespace
}  // namespace edf

extern "C" {

int edf_heads_split_rotary(void* stream, const void* x, const double* freq, const int32_t* positions, const void* wq,
                           const void* wk, void* q, void* k, void* v, long batch, long seq, int num_heads,
                           int num_kv_heads, int head_dim, int rotary_dim, int positions_per_row, int interleaved,
                           float eps, float amplitude, int dtype) {
  using namespace edf;
  RotaryArgs a{};
  a.x = (const char*)x, a.wq = (const char*)wq, a.wk = (const char*)wk, a.freq = freq, a.pos = positions;
  a.q = (char*)q, a.k = (char*)k, a.v = (char*)v;
  a.Hq = num_heads, a.Hkv = num_kv_heads, a.d = head_dim, a.rot = rotary_dim;
  a.pos_batch = positions_per_row ? (int)seq : 0, a.eps = eps, a.amp = amplitude;
  int rc = rotary_check(a, batch, seq, wk != nullptr, dtype);
  if (rc) return rc;
  a.tokens = batch * seq, a.T = (int)seq;
  unsigned wg = 0;
  return rotary_dispatch<false>(as_stream(stream), a, interleaved != 0, dtype, 1u << 30, &wg);
}

size_t edf_heads_split_rotary_backward_workspace_bytes(int head_dim) {
  return head_dim > 0 ? (size_t)edf::RO_BWD_WG * 2 * head_dim * sizeof(float) : 0;
}

int edf_heads_split_rotary_backward(void* stream, const void* x, const double* freq, const int32_t* positions,
                                    const void* wq, const void* wk, const void* grad_q, const void* grad_k,
                                    const void* grad_v, void* grad_x, void* grad_wq, void* grad_wk, void* workspace,
                                    size_t workspace_bytes, long batch, long seq, int num_heads, int num_kv_heads,
                                    int head_dim, int rotary_dim, int positions_per_row, int interleaved, float eps,
                                    float amplitude, int dtype) {
  using namespace edf;
  RotaryArgs a{};
  a.x = (const char*)x, a.wq = (const char*)wq, a.wk = (const char*)wk, a.freq = freq, a.pos = positions;
  a.q = (char*)const_cast<void*>(grad_q), a.k = (char*)const_cast<void*>(grad_k);
  a.v = (char*)const_cast<void*>(grad_v), a.dx = (char*)grad_x;
  a.Hq = num_heads, a.Hkv = num_kv_heads, a.d = head_dim, a.rot = rotary_dim;
  a.pos_batch = positions_per_row ? (int)seq : 0, a.eps = eps, a.amp = amplitude;
  int rc = rotary_check(a, batch, seq, wk != nullptr, dtype);
  if (rc) return rc;
  EDF_REQUIRE(grad_x && (!wq || (grad_wq && grad_wk)), EDF_ERR_INVALID_ARG, "null tensor pointer");
  if (wq) {
    const size_t need = edf_heads_split_rotary_backward_workspace_bytes(head_dim);
    EDF_REQUIRE(workspace && workspace_bytes >= need, EDF_ERR_WORKSPACE, "workspace too small: need %zu bytes", need);
    a.part = (float*)workspace;
  }
  a.tokens = batch * seq, a.T = (int)seq;
  hipStream_t s = as_stream(stream);
  unsigned wg = 0;
  rc = rotary_dispatch<true>(s, a, interleaved != 0, dtype, RO_BWD_WG, &wg);
  if (rc || !wq) return rc;
  const unsigned grid = (unsigned)((2 * head_dim + 15) / 16);
  if (dtype == EDF_BF16)
    rotary_dw_kernel<bf16><<<grid, 1024, 0, s>>>(a.part, (bf16*)grad_wq, (bf16*)grad_wk, (int)wg, head_dim);
  else
    rotary_dw_kernel<float><<<grid, 1024, 0, s>>>(a.part, (float*)grad_wq, (float*)grad_wk, (int)wg, head_dim);
  return check_launch("rotary norm weight gradient");
}

}  // extern "C"
