"""Attention over an 8-bit cache whose value scales lie far apart: a page of a large scale that has next to no weight takes
nothing from the others.

Tolerance, per element: P vs in two float16 parts (2^-22 of each, and 2^-39 of the query's largest) and 256 units of 2^-24 for
the float32 sums, of the sum of the terms' sizes, and half a step of the type of the result."""
import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce
from tests.test_gpu_cache8 import U, _pool, _to_gpu, bf16, f32

pytestmark = pytest.mark.gpu


def _check(q, caches, table, n, code, dtype):
    from edifice_amd import fused_scan as fs
    (kd, ks), (vd, vs) = (_to_gpu(*c, code) for c in caches)
    got = fs.paged_attention(q.to(dtype).cuda(), kd, vd, table.cuda(), n.cuda(), k_scale=ks, v_scale=vs).cpu().double()
    want, mag = od.paged_attention(q.to(dtype).double(), *(c * s[:, :, None, None] for c, s in caches), table, n)
    tol = (2.0 ** -22 + 256 * U) * mag + (2.0 ** -8 if dtype == bf16 else U) * want.abs()
    assert torch.isfinite(got).all()
    worst = float(((got - want).abs() / tol.clamp(min=1e-300)).max())
    assert worst <= 1, f"{worst:.3g} of the tolerance"


@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
@pytest.mark.parametrize("ratio", [24, 40])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("length, Hq, Hkv, d, block, code", [
    (64, 2, 1, 64, 16, "int8"),      # within a tile and past one
    (700, 4, 2, 128, 16, "e4m3"),    # a whole request, eight waves
    (3000, 8, 2, 128, 64, "int8"),   # in chunks
    (300, 3, 1, 256, 16, "e4m3"),    # tiles of 16 keys
    (200, 3, 1, 33, 5, "int8"),      # rows by element
])
def test_large_scale_with_little_weight(length, Hq, Hkv, d, block, code, place, ratio, dtype):
    """One page of values 2^ratio times the others', its keys' probabilities 2^(-2 ratio) times theirs."""
    announce("cache8 little weight", length=length, d=d, place=place, ratio=ratio, dtype=dtype)
    g = torch.Generator().manual_seed(length + ratio)
    caches, table, n = _pool((length,), Hkv, block, d, code, g)
    (kc, ks), (vc, vs) = caches
    pages = -(-length // block)
    page = int(table[0, {"first": 0, "middle": pages // 2, "last": pages - 1}[place]])
    q = torch.randn(1, Hq, d, generator=g)
    q[..., 0] = 16.0
    kc[..., 0] = 0.0
    down = 2 * ratio * 0.6931471805599453 * d ** 0.5 / 16  # what the first element takes from the page's scores
    for h in range(Hkv):
        if code == "int8":
            kc[page, h], ks[page, h] = torch.round(kc[page, h] * 0.1), down / 100
            kc[page, h, :, 0] = -100
        else:
            kc[page, h, :, 0], ks[page, h] = -256, down / 256
            kc[page, h, :, 1:] = 0.0
    ks[:] = ks.float().double()
    vs[page] *= 2.0 ** ratio
    _check(q, caches, table, n, code, dtype)


@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_scales_and_weights_of_every_size(code, dtype):
    """Value scales over 2^60 and scores over 30 beside one another, in no order; some pages of zeros."""
    announce("cache8 every size", code=code, dtype=dtype)
    g = torch.Generator().manual_seed(11)
    lengths = (900, 64, 33, 2500)
    caches, table, n = _pool(lengths, 2, 16, 64, code, g)
    (kc, ks), (vc, vs) = caches
    vs *= torch.exp2(torch.randint(-30, 31, vs.shape, generator=g).double())
    vs[torch.rand(vs.shape, generator=g) < 0.1] = 0.0
    q = torch.randn(len(lengths), 6, 64, generator=g) * torch.tensor([0.5, 2.0, 5.0, 5.0])[:, None, None]
    _check(q, caches, table, n, code, dtype)
