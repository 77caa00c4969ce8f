"""The plan of attention over packed texts without a GPU: the tests' restatement asks for the library's workspaces, and
every tile of every text comes up once in the order of work."""
import random

import pytest
import torch

from edifice_amd._native import lib
from tests import packed_plan as plan


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_workspaces_are_the_plans(dtype):
    L, rng, flag = lib(), random.Random(0), int(dtype == torch.bfloat16)
    ways = set()
    for _ in range(2000):
        Hkv = rng.choice([1, 2, 3, 8, 16])
        H, d = Hkv * rng.choice([1, 2, 3, 4, 8]), rng.randint(1, 128)
        N, M, texts = (int(2 ** rng.uniform(0, top)) for top in (16, 16, 10))
        if rng.random() < 0.05:
            M = (1 << 24) + rng.randint(-1, 1)
        sizes = H, Hkv, N, M, texts, d
        (way, parts), (kway, sums) = plan.queries(*sizes, dtype), plan.keys(*sizes, dtype)
        ways |= {("queries", way), ("keys", kway)}
        conf = H, Hkv, N, M, texts, d, 0, 0, flag
        assert L.edf_packed_attention_workspace_bytes(*conf) == parts(3), conf
        assert L.edf_packed_attention_backward_workspace_bytes(*conf) == -(-H * N * 4 // 256) * 256 + max(parts(0), sums), conf
    assert len(ways) == 6


@pytest.mark.parametrize("last_first", [True, False])
@pytest.mark.parametrize("m", [32, 64, 128])
def test_order_of_work_has_every_tile_once(m, last_first):
    rng = random.Random(m)
    for _ in range(12):
        sizes = [rng.choice([0, 1, m - 1, m, m + 1, rng.randint(0, 9 * m)]) for _ in range(rng.choice([1, 3, 40, 100, 255]))]
        if not sum(sizes):
            continue
        tiles = [-(-n // m) for n in sizes]
        got = [plan.tile_by_work(sizes, m, x, last_first) for x in range(sum(sizes) // m + len(sizes) + 1)]
        there = [t for t in got if t is not None]
        assert got[:len(there)] == there  # none after the last
        assert sorted(there) == [(s, i) for s, n in enumerate(tiles) for i in range(n)]
        # by what a tile has to walk, the most first: how far it is from its text's beginning, or from its end
        rank = [i if last_first else tiles[s] - 1 - i for s, i in there]
        assert rank == sorted(rank, reverse=True)
