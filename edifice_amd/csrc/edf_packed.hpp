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
  int hs;                // the four waves of a query workgroup take 2^hs heads of one key head, 128 >> hs queries of each
  int nx;                // tiles a head (an upper bound: which of them exist is known on the GPU)
  int by_work;           // tiles in order of their work, the longest first, rather than of the texts
  int chunks, len;       // queries: chunks of len key tiles; keys: shares of a key block's query tiles
  float scale, scale_log2;
};

constexpr int PK_M = 128;        // rows of a workgroup: queries of all its heads, or keys
constexpr int PK_ALL = 1 << 30;  // the window of a call without one
constexpr int PK_SORT = 256;     // texts, and the rows behind them, up to which tiles are put in order of work

// Tiles of m rows of `rows` rows in S texts: those of text s are numbered from offsets[s] / m + s on, the rows behind
// the last text are text S.  (Text s has at most floor(offsets[s + 1] / m) - floor(offsets[s] / m) + 1 of them.)
inline long packed_tiles(long rows, long texts, int m) { return rows / m + texts + 1; }

struct TextTile {
  int text, row0, n, first;  // the text, its first row and its rows; the tile's first row within the text (>= n: no tile)
};
EDF_DEVICE int text_begin(const int* off, int s, int rows) { return s == 0 ? 0 : min(max(off[s], 0), rows); }
EDF_DEVICE int text_end(const int* off, int S, int s, int rows, int begin) {
  return s >= S ? rows : max(text_begin(off, s + 1, rows), begin);
}
// tile x of 2^ms rows; all 64 lanes of a wave take part; the result is uniform
EDF_DEVICE TextTile find_tile(const int* off, int S, int rows, int ms, int x) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = S + 1;  // the text's number is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const bool at = s < hi && (text_begin(off, min(s, S), rows) >> ms) + s <= x;
    lo += (max((int)__popcll(__ballot(at)), 1) - 1) * step;
    hi = min(hi, lo + step);
  }
  TextTile t;
  t.text = __builtin_amdgcn_readfirstlane(lo);
  t.row0 = __builtin_amdgcn_readfirstlane(text_begin(off, t.text, rows));
  t.n = __builtin_amdgcn_readfirstlane(text_end(off, S, t.text, rows, t.row0)) - t.row0;
  t.first = (x - (t.row0 >> ms) - t.text) << ms;
  return t;
}
EDF_DEVICE int wave_sum_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// The same for S < PK_SORT with the tiles in another order: the x-th tile when those that are r-th from the end (last_first:
// from the start) of their text come before those that are (r - 1)-th.  A tile of queries sees the keys before it, a tile of
// keys is seen by the queries behind it, so that the longest work comes first, whichever text it is in.
// f(r) = sum over texts of max(0, tiles - r) tiles come before the r-th ones, of which a text with r tiles or more has one.
EDF_DEVICE TextTile find_tile_by_work(const int* off, int S, int rows, int ms, int x, bool last_first) {
  constexpr int C = PK_SORT / 64;
  const int lane = threadIdx.x & 63;
  int nb[C], begin[C], size[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int s = lane + 64 * c;
    begin[c] = s <= S ? text_begin(off, s, rows) : 0;
    size[c] = s <= S ? text_end(off, S, s, rows, begin[c]) - begin[c] : 0;
    nb[c] = (size[c] + (1 << ms) - 1) >> ms;
  }
  auto before = [&](int r) {
    int v = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) v += max(nb[c] - r, 0);
    return __builtin_amdgcn_readfirstlane(wave_sum_i(v));
  };
  TextTile t{0, 0, 0, 0};
  if (x >= before(0)) return t;  // past the last tile
  int lo = 0, hi = ((rows - 1) >> ms) + 1;  // before(lo) > x >= before(hi): no text has more than hi tiles
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before(mid) <= x) hi = mid;
    else lo = mid;
  }
  int rank = x - before(hi);  // among the texts with hi tiles or more, in their order
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const unsigned long long has = __ballot(nb[c] >= hi);
    const int count = __popcll(has);
    if (rank >= 0 && rank < count) {
      const unsigned long long me = __ballot((has >> lane) & 1 && __popcll(has & ((1ull << lane) - 1)) == rank);
      const int from = __builtin_ctzll(me);
      const int tiles = __builtin_amdgcn_readfirstlane(__shfl(nb[c], from));
      t.text = from + 64 * c;
      t.row0 = __builtin_amdgcn_readfirstlane(__shfl(begin[c], from));
      t.n = __builtin_amdgcn_readfirstlane(__shfl(size[c], from));
      t.first = (last_first ? hi - 1 : tiles - hi) << ms;
    }
    rank -= count;
  }
  return t;
}
// the rows of text s among `rows` (none behind the last text)
EDF_DEVICE void text_rows(const int* off, int S, int rows, int s, int& row0, int& n) {
  row0 = n = 0;
  if (s == S) return;
  row0 = __builtin_amdgcn_readfirstlane(text_begin(off, s, rows));
  n = __builtin_amdgcn_readfirstlane(text_end(off, S, s, rows, row0)) - row0;
}

// Workgroups of `groups` heads (or groups of heads) with `per` tiles each go round the eight XCDs.  A head's tiles, which
// share its keys, stay on as few of them as give every XCD the same share of each part of the tiles' order, in which work
// falls: one where there are a multiple of eight heads, 8 / groups of them for 1, 2 or 4 heads, all for any other number.
inline long packed_grid(long groups, long per) {
  return groups % 8 != 0 && 8 % groups == 0 ? 8 * ((per * groups + 7) / 8) : groups * per;
}
// the head and tile of this workgroup; false: none
EDF_DEVICE bool packed_block(int groups, int per, int& x, int& grp) {
  const int id = blockIdx.x, c = id & 7, k = id >> 3;
  if ((groups & 7) == 0) {
    grp = c * (groups >> 3) + k / per;
    x = k % per;
  } else if (groups == 1 || groups == 2 || groups == 4) {
    const int share = 8 / groups;
    grp = c / share;
    x = k * share + c % share;
  } else {
    grp = id % groups;
    x = id / groups;
  }
  return x < per;
}

// The key tiles of a block of m queries from position q0 on, as KeyTiles has them; none where the block lies before its keys.
template <int BN>
struct BlockTiles {
  int ns, edge, ne, diag, nd, mid, count, first_whole;
  EDF_DEVICE BlockTiles(int q0, int m, int T, int W, int S) {
    if (q0 + m <= 0) T = 0;
    const int end = (max(0, min(T, q0 + m)) + BN - 1) / BN;
    const int wt0 = min(max(0, q0 - W + 1) / BN, end);  // first tile of the window
    ns = min((min(S, T) + BN - 1) / BN, wt0);
    const int past = q0 + m - 1 - W;  // keys up to here are hidden from the last query
    mid = min(max(past < 0 ? 0 : past / BN + 1, wt0), end);
    edge = wt0;
    ne = mid - wt0;
    diag = max(min(max(0, q0 + 1) / BN, end), mid);
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

// What a workgroup of queries works on: four waves, each 32 queries of one head at positions pw .. pw + 31 of the text's nk
// keys, and the workgroup's chunk [t0, t1) of their key tiles.
template <int BN>
struct QueryTile {
  int head, kvhead, myq, nq, pw, nk, chunk, t0, t1;  // head, myq (query within the text), pw: of the wave or lane
  long row0, krow;                                   // rows of the text's first query (of the wave's head) and key
  bool none;
  BlockTiles<BN> kt;
  EDF_DEVICE static TextTile tile(const PackArgs& a, int x) {
    const int ms = 7 - a.hs;
    return a.by_work ? find_tile_by_work(a.qo, a.S, a.N, ms, x, true) : find_tile(a.qo, a.S, a.N, ms, a.nx - 1 - x);
  }
  EDF_DEVICE QueryTile(const PackArgs& a) : kt(0, 0, 0, 1, 0) {
    const int w = threadIdx.x >> 6, li = threadIdx.x & 31, wu = __builtin_amdgcn_readfirstlane(w);
    int x, grp;
    none = !packed_block(a.H >> a.hs, a.nx * a.chunks, x, grp);
    if (none) return;
    chunk = x % a.chunks;
    const TextTile t = tile(a, x / a.chunks);
    head = (grp << a.hs) + (wu & ((1 << a.hs) - 1));
    kvhead = (grp << a.hs) / a.G;
    nq = t.n;
    none = t.first >= nq;
    int key0;
    text_rows(a.ko, a.S, a.M, t.text, key0, nk);
    const int wq = t.first + 32 * (w >> a.hs);  // the wave's first query
    myq = wq + li;
    pw = wq + nk - nq;
    row0 = (long)head * a.N + t.row0;
    krow = (long)kvhead * a.M + key0;
    kt = BlockTiles<BN>(t.first + nk - nq, PK_M >> a.hs, nk, a.W, a.sinks);
    t0 = min(chunk * a.len, kt.count);
    t1 = min(t0 + a.len, kt.count);
    if (chunk > 0 && t0 >= kt.count) none = true;  // the first chunk answers for a tile without keys
  }
  EDF_DEVICE int key0(int t) const { return kt.key0(t0 + t); }
  // some query of the wave sees a key of the bn keys from k0 on
  EDF_DEVICE bool visible(const PackArgs& a, int k0, int bn) const {
    return (k0 <= pw + 31 && k0 + bn + a.W > pw + 1) || k0 < a.sinks;
  }
};

// Tiles in order of their work where they are some rounds of the GPU's 512 places, so that the last ones to start count, and
// texts are long enough (128 keys on average) that a workgroup's search for its tile does not.
inline bool order_by_work(const PackArgs& a, long wgs) {
  return wgs > 512 && wgs <= 4096 && a.S < PK_SORT && a.M >= 128L * a.S;
}

// heads of a query workgroup: as many of a key head's as the four waves take
inline int head_shift(int G) { return G % 4 == 0 ? 2 : G % 2 == 0 ? 1 : 0; }
// How the key tiles (of BN) of a query workgroup are cut: into chunks of `len` tiles where the call's workgroups without it
// would not fill the GPU's 512 places.  The longest text may have all keys, so the grid has a chunk for each part of those,
// most of which find no tile.
inline void query_plan(PackArgs& a, int BN) {
  a.hs = head_shift(a.G);
  const int m = PK_M >> a.hs;
  a.nx = (int)packed_tiles(a.N, a.S, m);
  a.chunks = 1, a.len = 1 << 30;
  const long wgs = (long)(a.H >> a.hs) * a.nx;
  a.by_work = order_by_work(a, wgs);
  if (wgs >= 512) return;
  long keys = a.M;
  if (a.W < PK_ALL) keys = std::min(keys, (long)a.W + m + a.sinks + 2L * BN);
  const long most = (keys + BN - 1) / BN + 1, want = std::min(32L, std::max(1L, 4096 / wgs));
  const long len = std::max(4L, (most + want - 1) / want);
  a.chunks = (int)((most + len - 1) / len);
  if (a.chunks > 1) a.len = (int)len;
}
inline size_t chunk_bytes(const PackArgs& a, int extra) {  // extra: floats a row beside the padded head
  return a.chunks == 1 ? 0 : (size_t)a.chunks * a.H * a.N * (window_pad(a.d) + extra) * sizeof(float);
}
constexpr int key_tile(int dtype) { return dtype == EDF_BF16 ? 64 : 32; }

int packed_check(int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim, int window, int sinks,
                 int dtype);

}  // namespace edf
