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
  float *part, *ml;      // queries: [head group][item][128] unnormalised outputs (or dQ) of chunks; ml: maxima, two sums;
                         // keys: part [Hkv][item] dK and dV of chunks
  int* plan;             // [head group][tile] first item and number of chunks
  const int *qo, *ko;
  int N, M, S, H, G, d, W, sinks;
  int hs;                // the four waves of a query workgroup take 2^hs heads of one key head, 128 >> hs queries of each
  int nx;                // tiles a head (an upper bound: which of them exist is known on the GPU)
  int by_work;           // tiles in order of their work, the longest first, rather than of the texts
  int items;             // chunks a head group (an upper bound), 0: the other tensor's tiles are not cut
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
  int other0, m;             // its first row and rows in the other tensor (none behind the last text)
};
EDF_DEVICE int text_begin(const int* off, int s, int rows) { return s == 0 ? 0 : min(max(off[s], 0), rows); }
EDF_DEVICE int text_end(const int* off, int S, int s, int rows, int begin) {
  return s >= S ? rows : max(text_begin(off, s + 1, rows), begin);
}
// the rows of text s in the other tensor
EDF_DEVICE void other_rows(const int* off, int S, int rows, TextTile& t) {
  t.other0 = t.m = 0;
  if (t.text == S) return;
  t.other0 = __builtin_amdgcn_readfirstlane(text_begin(off, t.text, rows));
  t.m = max(__builtin_amdgcn_readfirstlane(text_begin(off, t.text + 1, rows)) - t.other0, 0);
}
// tile x of 2^ms rows, of the last text that can have it; all 64 lanes of a wave take part; the result is uniform
EDF_DEVICE TextTile find_tile(const int* off, int rows, const int* off2, int rows2, int S, int ms, int x) {
  const int lane = threadIdx.x & 63;
  TextTile t;
  if (S < 64) {  // a lane a text: all offsets in one load
    const int s = min(lane, S), b = text_begin(off, s, rows), e = text_end(off, S, s, rows, b);
    const int b2 = s == S ? 0 : text_begin(off2, s, rows2), e2 = s == S ? 0 : max(text_begin(off2, s + 1, rows2), b2);
    const int from = 63 - __builtin_clzll(__ballot(lane <= S && (b >> ms) + lane <= x));  // text 0 begins at 0
    t.text = from;
    t.row0 = __builtin_amdgcn_readlane(b, from);
    t.n = __builtin_amdgcn_readlane(e, from) - t.row0;
    t.other0 = __builtin_amdgcn_readlane(b2, from);
    t.m = __builtin_amdgcn_readlane(e2, from) - t.other0;
  } else {
    int lo = 0, hi = S + 1;  // the text's number is in [lo, hi)
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, s = lo + lane * step;
      const bool at = s < hi && (text_begin(off, min(s, S), rows) >> ms) + s <= x;  // so for lo
      lo += (63 - __builtin_clzll(__ballot(at))) * step;
      hi = min(hi, lo + step);
    }
    t.text = __builtin_amdgcn_readfirstlane(lo);
    t.row0 = __builtin_amdgcn_readfirstlane(text_begin(off, t.text, rows));
    t.n = __builtin_amdgcn_readfirstlane(text_end(off, S, t.text, rows, t.row0)) - t.row0;
    other_rows(off2, S, rows2, t);
  }
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
EDF_DEVICE TextTile find_tile_by_work(const int* off, int rows, const int* off2, int rows2, int S, int ms, int x,
                                      bool last_first) {
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
  TextTile t{0, 0, 0, 0, 0, 0};
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
  other_rows(off2, S, rows2, t);
  return t;
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

// Where queries (or keys) are few against the GPU the key (or query) tiles that each of their tiles walks are cut into chunks,
// an item of work each.  All workgroups of a call come to the same plan from the offsets alone: chunks of len tiles, so that
// they and the tiles' last, shorter ones are as many as the GPU's places (a chunk more than those waits for a whole one to
// end), numbered from tile to tile.  Item `item` of a head group's; threads look at two tiles of 2^ms rows each, of which
// there are fewer than 512; count(first, n, m): the tiles that the one from row `first` on walks.
// Queries uncut, and cut: 8 texts of up to 64 queries on 28563 keys, 32(8)x128, 80 and 44 us; 247 queries on 30000 keys 550
// and 147.  Keys (forward and backward) with an equal number of shares of each block's query tiles, and with such chunks: 8
// texts to 2000, 8(4)x128, 244 and 175 us, one of 4000, 16(4)x128, 548 and 420, 4 to 1500, 32(8)x128, 262 and 191, 12 to 4096,
// 8(1)x128, 1189 and 700; float32 8 to 2000, 8(4)x64, 636 and 450.  As many chunks as 576 to 1536 places are slower at most of
// these, and a search for the shortest len costs 1 to 4 us more than it saves.
constexpr int PK_ITEMS = 512, PK_PLAN = 512;
struct Item {
  TextTile tile;
  int x, chunk, chunks, len;  // the tile's number, which of its chunks, how many, tiles of one
  bool none;
};
template <typename Count>
EDF_DEVICE Item find_item(const int* off, int rows, const int* off2, int rows2, int S, int ms, int groups, int least,
                          int item, int* lds, Count tiles) {
  const int tid = threadIdx.x, lane = tid & 63;
  int *so = lds, *sk = lds + PK_PLAN + 2, *sum = sk + PK_PLAN + 2, *found = sum + 8;
  for (int s = tid; s <= S; s += 256) {
    so[s] = text_begin(off, s, rows);
    sk[s] = text_begin(off2, s, rows2);
  }
  if (tid == 0) {
    so[S + 1] = rows;
    found[0] = -1;
  }
  __syncthreads();
  int count[2], text[2], chunks[2];
  int mine = 0, there = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int x = 2 * tid + i;
    count[i] = -1, text[i] = 0;
    if (x >= (rows >> ms) + S + 1) continue;
    int lo = 0, hi = S + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((so[mid] >> ms) + mid <= x) lo = mid;
      else hi = mid;
    }
    text[i] = lo;
    const int n = max(so[lo + 1] - so[lo], 0), first = (x - (so[lo] >> ms) - lo) << ms;
    if (first >= n) continue;
    count[i] = tiles(first, n, lo < S ? max(sk[lo + 1] - sk[lo], 0) : 0);
    mine += count[i];
    ++there;
  }
  const int ws = wave_sum_i(mine), wt = wave_sum_i(there);
  if (lane == 0) {
    sum[tid >> 6] = ws;
    sum[4 + (tid >> 6)] = wt;
  }
  __syncthreads();
  const long all = (long)sum[0] + sum[1] + sum[2] + sum[3];
  // a tile's last chunk is half a chunk on average
  const int parts = max(PK_ITEMS - (sum[4] + sum[5] + sum[6] + sum[7]) * groups / 2, PK_ITEMS / 2);
  const int len = (int)max((long)least, (all * groups + parts - 1) / parts);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) chunks[i] = count[i] < 0 ? 0 : max(1, (count[i] + len - 1) / len);
  int incl = chunks[0] + chunks[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(incl, o);
    incl += lane >= o ? up : 0;
  }
  if (lane == 63) sum[4 + (tid >> 6)] = incl;
  __syncthreads();
  int at = incl - chunks[0] - chunks[1];  // items before this thread's tiles
  for (int w = 0; w < (tid >> 6); ++w) at += sum[4 + w];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (item >= at && item < at + chunks[i]) {
      found[0] = 2 * tid + i;
      found[1] = text[i];
      found[2] = item - at;
      found[3] = chunks[i];
    }
    at += chunks[i];
  }
  __syncthreads();
  Item t;
  t.x = __builtin_amdgcn_readfirstlane(found[0]);
  t.none = t.x < 0;
  const int s = __builtin_amdgcn_readfirstlane(found[1]);
  if (t.none) return t;
  t.tile.text = s;
  t.tile.row0 = __builtin_amdgcn_readfirstlane(so[s]);
  t.tile.n = __builtin_amdgcn_readfirstlane(max(so[s + 1] - so[s], 0));
  t.tile.first = (t.x - (t.tile.row0 >> ms) - s) << ms;
  t.tile.other0 = s < S ? __builtin_amdgcn_readfirstlane(sk[s]) : 0;
  t.tile.m = s < S ? __builtin_amdgcn_readfirstlane(max(sk[s + 1] - sk[s], 0)) : 0;
  t.chunk = __builtin_amdgcn_readfirstlane(found[2]);
  t.chunks = __builtin_amdgcn_readfirstlane(found[3]);
  t.len = __builtin_amdgcn_readfirstlane(len);
  __syncthreads();  // the caller's tiles go into the same memory
  return t;
}

// What a workgroup of queries works on: four waves, each 32 queries of one head at positions pw .. pw + 31 of the text's nk
// keys, and the workgroup's chunk [t0, t1) of their key tiles.
template <int BN>
struct QueryTile {
  int head, kvhead, myq, nq, pw, nk, t0, t1;  // head, myq (query within the text), pw: of the wave or lane
  long row0, krow;                            // rows of the text's first query (of the wave's head) and key
  long slot;                                  // of one of several chunks: this lane's row of part and ml, or -1
  bool none, first;                           // first: the tile's first chunk
  BlockTiles<BN> kt;
  // lds: 4 KB and some that the kernel uses later
  EDF_DEVICE QueryTile(const PackArgs& a, void* lds) : kt(0, 0, 0, 1, 0) {
    const int w = threadIdx.x >> 6, li = threadIdx.x & 31, wu = __builtin_amdgcn_readfirstlane(w);
    const int groups = a.H >> a.hs, ms = 7 - a.hs;
    int x, grp, chunk = 0, len = 0;
    none = !packed_block(groups, a.items > 0 ? a.items : a.nx, x, grp);
    if (none) return;
    TextTile t;
    slot = -1;
    if (a.items > 0) {
      const Item it = find_item(a.qo, a.N, a.ko, a.M, a.S, ms, groups, 4, x, (int*)lds, [&](int first, int n, int m) {
        return BlockTiles<BN>(first + m - n, 1 << ms, m, a.W, a.sinks).count;
      });
      none = it.none;
      if (none) return;
      t = it.tile, chunk = it.chunk, len = it.len;
      if (it.chunks > 1) slot = ((long)grp * a.items + x) * PK_M + 32 * w + li;
      if (chunk == 0 && threadIdx.x == 0) {
        int* p = a.plan + 2 * ((long)grp * a.nx + it.x);
        p[0] = x;
        p[1] = it.chunks;
      }
    } else {
      t = a.by_work ? find_tile_by_work(a.qo, a.N, a.ko, a.M, a.S, ms, x, true)
                    : find_tile(a.qo, a.N, a.ko, a.M, a.S, ms, a.nx - 1 - x);
      none = t.first >= t.n;
      if (none) return;
    }
    head = (grp << a.hs) + (wu & ((1 << a.hs) - 1));
    kvhead = (grp << a.hs) / a.G;
    nq = t.n, nk = t.m;
    const int wq = t.first + 32 * (w >> a.hs);  // the wave's first query
    myq = wq + li;
    pw = wq + nk - nq;
    row0 = (long)head * a.N + t.row0;
    krow = (long)kvhead * a.M + t.other0;
    kt = BlockTiles<BN>(t.first + nk - nq, PK_M >> a.hs, nk, a.W, a.sinks);
    first = chunk == 0;
    t0 = chunk * len;
    t1 = a.items > 0 ? min(t0 + len, kt.count) : kt.count;
  }
  EDF_DEVICE int key0(int t) const { return kt.key0(t0 + t); }
  // some query of the wave sees a key of the bn keys from k0 on
  EDF_DEVICE bool visible(const PackArgs& a, int k0, int bn) const {
    return (k0 <= pw + 31 && k0 + bn + a.W > pw + 1) || k0 < a.sinks;
  }
};

// One row of a query tile in chunks, for the kernels that join them: LANES lanes a row, 256 / LANES rows a workgroup.
template <int LANES>
struct ChunkRow {
  static constexpr int PIECES = PK_M * LANES / 256;  // workgroups a tile
  int chunks;      // 0: nothing to do
  long row, slot;  // of the outputs; of part and ml, the first chunk's
  EDF_DEVICE ChunkRow(const PackArgs& a) : chunks(0) {
    int x, grp;
    if (!packed_block(a.H >> a.hs, a.nx * PIECES, x, grp)) return;
    const int ms = 7 - a.hs, r = x % PIECES * (256 / LANES) + threadIdx.x / LANES;
    const TextTile t = find_tile(a.qo, a.N, a.ko, a.M, a.S, ms, x / PIECES);
    const int q = t.first + 32 * (r >> 5 >> a.hs) + (r & 31);
    if (t.first >= t.n || q >= t.n) return;
    const int* p = a.plan + 2 * ((long)grp * a.nx + x / PIECES);
    const int item = p[0], n = p[1];
    if (n <= 1 || item < 0 || n > a.items - item) return;  // one chunk, or no plan (offsets that do not ascend)
    chunks = n;
    row = (long)((grp << a.hs) + ((r >> 5) & ((1 << a.hs) - 1))) * a.N + t.row0 + q;
    slot = ((long)grp * a.items + item) * PK_M + r;
  }
};

// Tiles in order of their work where they are some rounds of the GPU's 512 places, so that the last ones to start count, and
// texts are long enough (128 keys on average) that a workgroup's search for its tile does not.  In the texts' order, and in
// that of work: dK and dV of 12 texts to 4096, 32(8)x128, 1451 and 1209 us; forward of 3 texts to 10000, 16(2)x64, 302 and
// 286; of 8 texts to 4096, 8x128, 173 and 153.  Past 4096 workgroups the two are even.
inline bool order_by_work(const PackArgs& a, long wgs) {
  return wgs > 512 && wgs <= 4096 && a.S < PK_SORT && a.M >= 128L * a.S;
}

// Heads of a query workgroup: as many of a key head's as the four waves take, since they read its keys once and few queries
// of a text fill the waves all the same.  One head a workgroup, and four: 8 texts of up to 64 queries on 28563 keys, 32(8)x128,
// 152 and 80 us (before chunks); 200 texts of 150 tokens, 16(4)x64, forward and backward 302 and 253.
inline int head_shift(int G) { return G % 4 == 0 ? 2 : G % 2 == 0 ? 1 : 0; }
// Tiles are cut where the call's workgroups would not fill the GPU's 512 places, and keys are enough that chunks are worth the
// kernel that joins them: one text, 8(4)x64, cut and uncut, bf16 of 300 keys 14.3 and 9.7 us, 500 14.7 and 13.1, 1000 15.9 and
// 18.8; float32 of 150 keys 20.2 and 16.1, 250 20.3 and 23.9.  A tile has a chunk for each len of its key tiles and one for
// the rest, so there are at most PK_ITEMS over all groups and one a tile.
inline void query_plan(PackArgs& a, int BN) {
  a.hs = head_shift(a.G);
  a.nx = (int)packed_tiles(a.N, a.S, PK_M >> a.hs);
  const long groups = a.H >> a.hs, wgs = groups * a.nx;
  a.by_work = order_by_work(a, wgs);
  // (the plan's sum of key tiles is an int: 2^24 keys of 512 tiles)
  const bool cut = wgs < PK_PLAN && a.M > (BN == 64 ? 512 : 192) && a.M < (1 << 24);
  a.items = cut ? (int)((PK_ITEMS + groups - 1) / groups) + a.nx : 0;
}
inline size_t chunk_bytes(const PackArgs& a, int extra) {  // extra: floats a row beside the padded head
  const size_t groups = a.H >> a.hs;
  return a.items == 0 ? 0
                      : groups * a.items * PK_M * (window_pad(a.d) + extra) * sizeof(float) + groups * a.nx * 2 * sizeof(int);
}
inline void chunk_memory(PackArgs& a, float* part, int extra) {
  const size_t rows = (size_t)(a.H >> a.hs) * a.items * PK_M;
  a.part = part, a.ml = part + rows * window_pad(a.d);
  a.plan = (int*)(a.ml + rows * extra);
}
constexpr int key_tile(int dtype) { return dtype == EDF_BF16 ? 64 : 32; }

int packed_check(int num_heads, int num_kv_heads, long rows, long key_rows, int texts, int head_dim, int window, int sinks,
                 int dtype);

}  // namespace edf
