"""GPU parity of attention over packed texts, forward and backward, on each way in which it divides its work: tiles in order
of work, in the texts' order, and in chunks (tests/packed_plan.py says which way a case takes; the tolerances are those of
tests/test_gpu_packed_attention.py)."""
import random

import pytest
import torch

from tests import packed_plan as plan
from tests.test_gpu_packed_attention import _name, bf16, f32, test_packed_attention_fwd_bwd as check

pytestmark = pytest.mark.gpu

WIDTHS = [(20, bf16), (32, bf16), (64, bf16), (80, bf16), (96, bf16), (112, bf16), (128, bf16), (30, f32), (64, f32), (96, f32),
          (128, f32)]
LONG = (700, 1, 333, 0, 256, 512, 129, 90, 610, 569)              # 3200 rows
MANY = tuple(n for pair in zip(LONG, (0, 1, 2, 3, 0, 5, 40, 31, 1, 33)) for n in pair) + (1, 0, 2, 7, 128, 1, 0, 1, 2, 4, 0, 9)


@pytest.mark.parametrize("d, dtype", WIDTHS, ids=str)
def test_tiles_in_order_of_work(d, dtype):
    """Texts of several hundred tokens with shared key heads, none cut: an empty text, rows behind, a window at some widths."""
    window, sinks = ((0, 0), (300, 5))[d // 32 % 2]
    case = LONG, None, 9, 32, 16, d, window, sinks, dtype
    assert plan.of_case(case) == ("by work", "by work")
    check(case)


@pytest.mark.parametrize("d, dtype", WIDTHS, ids=str)
def test_tiles_in_order_of_texts(d, dtype):
    window, sinks = ((300, 5), (0, 0))[d // 32 % 2]
    case = MANY, None, 9, 32, 16, d, window, sinks, dtype
    assert plan.of_case(case) == ("by text", "by text")
    check(case)


def _ragged(texts, mean, seed):
    rng = random.Random(seed)
    return tuple(rng.choice([0, 1, rng.randint(1, 2 * mean), rng.randint(1, 4 * mean), 3 * mean]) for _ in range(texts))


@pytest.mark.parametrize("case, ways", [
    # more texts than a load of 64 offsets has
    ((_ragged(100, 120, 1), None, 0, 4, 4, 64, 0, 0, bf16), ("by work", "by work")),
    ((_ragged(130, 120, 2), None, 70, 4, 4, 128, 0, 0, bf16), ("by work", "by work")),
    ((_ragged(255, 120, 3), None, 3, 2, 2, 32, 50, 2, f32), ("by work", "by work")),
    # heads of four in a workgroup: queries alone
    ((LONG[:7], None, 0, 32, 8, 128, 0, 0, bf16), ("by work", "cut")),
    # conversations that go on: few queries at the end of longer keys, more workgroups than places
    ((tuple(i % 5 for i in range(64)), tuple(140 + 9 * i % 400 for i in range(64)), 0, 32, 8, 128, 0, 0, bf16),
     ("by work", "by work")),
    ((tuple(1 + i % 3 for i in range(66)), tuple(130 + 11 * i % 300 for i in range(66)), 5, 32, 8, 64, 100, 3, bf16),
     ("by work", "by work")),
    ((tuple(1 + i % 40 for i in range(40)), tuple(130 + 31 * i % 300 for i in range(40)), 0, 16, 16, 64, 0, 0, f32),
     ("by work", "by work")),
    # more queries than keys in some texts
    ((tuple(3 * i for i in range(20)), tuple(60 * (20 - i) for i in range(20)), 1, 32, 32, 64, 0, 0, bf16),
     ("by work", "by work")),
    # chunks of more texts than threads look up at once
    ((_ragged(300, 4, 4), None, 6, 4, 1, 128, 0, 0, bf16), ("cut", "cut")),
    ((_ragged(400, 3, 5), None, 0, 1, 1, 64, 0, 0, bf16), ("cut", "cut")),
    ((_ragged(300, 3, 6), None, 2, 1, 1, 96, 9, 2, f32), ("cut", "cut")),
    ((tuple(i % 3 for i in range(280)), _ragged(280, 20, 7), 0, 1, 1, 64, 0, 0, f32), ("cut", "cut")),
], ids=lambda c: f"{len(c[0])}texts{sum(c[0])}of{sum(c[1] or c[0])}-" + _name(((), None) + c[2:])[1:] if len(c) > 2 else "-".join(c))
def test_many_texts_and_long_keys(case, ways):
    assert plan.of_case(case) == ways
    check(case)
