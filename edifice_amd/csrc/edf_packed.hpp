// Shared by the forward and backward of causal attention over packed texts: the arguments, and how a workgroup finds the
// text and tile that it works on.
//
// Text s has queries rows qo[s] .. qo[s + 1] - 1 of [H, N, d] and keys rows ko[s] .. ko[s + 1] - 1 of [Hkv, M, d]; query i
// of n stands at position i + m - n among its m keys.  Offsets are read on the GPU, so that a captured call may be replayed
// with other lengths, and clamped, so that none leads out of the tensors.
#pragma once

#include "edf_window.hpp"

namespace edf {

struct PackArgs {
  const void *q, *k, *v, *o, *go;
  void *out, *dq, *dk, *dv;
  float *lse, *dd;       // [H N]
  float *part, *ml;      // forward: [chunk][H N] unnormalised outputs of chunks of keys, their maxima and sums;
                         // backward: part [chunk][Hkv M / 128 ...] dK and dV of chunks of queries
  const int *qo, *ko;
  int N, M, S, H, G, d, W, sinks;
  int nx;                // tiles a head (an upper bound: which of them exist is known on the GPU)
  int chunks, len;       // forward: chunks of len key tiles; backward: shares of a key block's query tiles
  float scale, scale_log2;
};

constexpr int PK_M = 128;       // queries, or keys in the backward, of a workgroup
constexpr int PK_ALL = 1 << 30;  // the window of a call without one

// Tiles of PK_M rows of `rows` rows in S texts: those of text s are numbered from offsets[s] / PK_M + s on, the rows behind
// the last text are text S.  (Text s has at most floor(offsets[s + 1] / PK_M) - floor(offsets[s] / PK_M) + 1 of them.)
inline long packed_tiles(long rows, long texts) { return rows / PK_M + texts + 1; }

struct TextTile {
  int text, row0, n, first;  // the text, its first row and its rows; the tile's first row within the text (>= n: no tile)
};
EDF_DEVICE int text_begin(const int* off, int s, int rows) { return s == 0 ? 0 : min(max(off[s], 0), rows); }
// all 64 lanes of a wave take part; the result is uniform
EDF_DEVICE TextTile find_tile(const int* off, int S, int rows, int x) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = S + 1;  // the text's number is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const bool at = s < hi && text_begin(off, min(s, S), rows) / PK_M + s <= x;
    lo += (max((int)__popcll(__ballot(at)), 1) - 1) * step;
    hi = min(hi, lo + step);
  }
  TextTile t;
  t.text = __builtin_amdgcn_readfirstlane(lo);
  t.row0 = __builtin_amdgcn_readfirstlane(text_begin(off, t.text, rows));
  const int end = t.text == S ? rows : __builtin_amdgcn_readfirstlane(text_begin(off, t.text + 1, rows));
  t.n = max(end - t.row0, 0);
  t.first = (x - t.row0 / PK_M - t.text) * PK_M;
  return t;
}
// the rows of text s among `rows` (none behind the last text)
EDF_DEVICE void text_rows(const int* off, int S, int rows, int s, int& row0, int& n) {
  row0 = n = 0;
  if (s == S) return;
  row0 = __builtin_amdgcn_readfirstlane(text_begin(off, s, rows));
  n = max(__builtin_amdgcn_readfirstlane(text_begin(off, s + 1, rows)) - row0, 0);
}

// the (tile, head) of logical workgroup id, the tiles of a head on one XCD
EDF_DEVICE void packed_block(const PackArgs& a, int per_head, int& x, int& head) {
  const int id = remap_xcd(blockIdx.x, gridDim.x);
  x = id % per_head;
  head = id / per_head;
}

int packed_check(int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim, int window, int sinks,
                 int dtype);

}  // namespace edf
