"""The 8-bit cache's write where the slots of a page do not follow one another, exactly the definition's numbers and scales:
the tokens of a page follow one another in a row, their slots are any of the page's, in any order."""
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_cache8 import _random_cache, _write_both, bf16, f32

pytestmark = pytest.mark.gpu


def _values(B, Hkv, T, d, dtype, g):
    return [(torch.randn(B, Hkv, T, d, generator=g) * torch.exp2(torch.randint(-6, 14, (B, Hkv, T, 1), generator=g).float()))
            .to(dtype) for _ in range(2)]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("slots", [[0, 2], [1, 3], [3, 1, 0], [2, 3, 0, 1], [5, 7, 0, 3, 2, 9]], ids=str)
def test_a_few_tokens_of_a_page(slots, code):
    announce("cache8 slots", slots=slots, code=code)
    g = torch.Generator().manual_seed(len(slots))
    caches = [_random_cache(3, 2, 4, 16, code, g) for _ in range(2)]
    _write_both(_values(1, 2, len(slots), 16, f32, g), [slots], caches, code, f32)


def _any_slots(T, block, pages, g):
    """T slots, page by page: of each some, all of them in order, the last ones in order, or all in any order."""
    slots = []
    while len(slots) < T:
        page = pages.pop()
        kind = int(torch.randint(0, 4, (1,), generator=g))
        n = int(torch.randint(1, block + 1, (1,), generator=g))
        offs = torch.randperm(block, generator=g)[:n].tolist()
        offs = [offs, list(range(block)), list(range(block - n, block)), torch.randperm(block, generator=g).tolist()][kind]
        slots += [page * block + o for o in offs]
    return slots[:T]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("B, Hkv, T, d, block, dtype", [
    (2, 2, 200, 16, 8, bf16),
    (3, 1, 150, 64, 16, f32),
    (1, 2, 400, 24, 100, bf16),     # a page's tokens across 64 of them
    (2, 1, 300, 32, 64, bf16),
    (1, 1, 500, 64, 200, f32),      # four waves a page
    (1, 2, 260, 33, 130, f32),      # and by element
    (2, 2, 70, 7, 5, bf16),
    (2, 1, 90, 128, 32, bf16),
])
def test_any_order(B, Hkv, T, d, block, dtype, code):
    announce("cache8 slots in any order", T=T, d=d, block=block, code=code)
    g = torch.Generator().manual_seed(T + d)
    blocks = B * T
    pages = torch.randperm(blocks, generator=g).tolist()
    slots = [_any_slots(T, block, pages, g) for _ in range(B)]
    slots[-1][T - 3:] = [-1] * 3  # and padding behind
    caches = [_random_cache(blocks, Hkv, block, d, code, g) for _ in range(2)]
    _write_both(_values(B, Hkv, T, d, dtype, g), slots, caches, code, dtype)
