"""How attention over packed texts divides its work, restated for the tests that have to reach each way: the rules of
edifice_amd/csrc/edf_packed.hpp (query_plan, order_by_work) and packed_attn_bwd.hip (backward_plan) on sizes alone."""
import torch

TILE, PLACES = 128, 512


def _tiles(rows, texts, m):
    return rows // m + texts + 1


def _pad(d):
    return -(-d // 32) * 32


def _by_work(wgs, texts, keys):
    return PLACES < wgs <= 4096 and texts < 256 and keys >= 128 * texts


def queries(H, Hkv, N, M, texts, d, dtype):
    """(way, bytes of a chunk's outputs and of the plan without the sums): "cut", "by work" or "by text"."""
    G = H // Hkv
    share = 4 if G % 4 == 0 else 2 if G % 2 == 0 else 1
    groups, nx = H // share, _tiles(N, texts, TILE // share)
    wgs = groups * nx
    if wgs < PLACES and M > (512 if dtype == torch.bfloat16 else 192) and M < 1 << 24:
        items = -(-PLACES // groups) + nx
        return "cut", lambda extra: groups * items * TILE * (_pad(d) + extra) * 4 + groups * nx * 8
    return "by work" if _by_work(wgs, texts, M) else "by text", lambda extra: 0


def keys(H, Hkv, N, M, texts, d, dtype):
    nx, rows = _tiles(M, texts, TILE), N * (H // Hkv)
    wgs = Hkv * nx
    if wgs < PLACES and (512 if dtype == torch.bfloat16 else 64) < rows < 1 << 25 and M < 1 << 24:
        items = -(-PLACES // Hkv) + nx
        return "cut", Hkv * items * 2 * TILE * _pad(d) * 4 + Hkv * nx * 8
    return "by work" if _by_work(wgs, texts, M) else "by text", 0


def of_case(case):
    """The ways of a test's (query lengths, key lengths or None, rows behind, Hq, Hkv, d, window, sinks, dtype)."""
    nq, nk, behind, H, Hkv, d, _, _, dtype = case
    sizes = H, Hkv, sum(nq) + behind, sum(nk or nq) + behind, len(nq), d, dtype
    return queries(*sizes)[0], keys(*sizes)[0]


def tile_by_work(sizes, m, x, last_first):
    """The x-th tile of m rows (text, which of its tiles) of texts of these sizes, in order of work, as find_tile_by_work
    comes to it; None past the last."""
    tiles = [-(-n // m) for n in sizes]
    before = lambda r: sum(max(t - r, 0) for t in tiles)  # noqa: E731
    if x >= before(0):
        return None
    lo, hi = 0, (sum(sizes) - 1) // m + 1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (lo, mid) if before(mid) <= x else (mid, hi)
    text = [s for s, t in enumerate(tiles) if t >= hi][x - before(hi)]
    return text, hi - 1 if last_first else tiles[text] - hi
