"""The 8-bit cache's write, exactly the definition's numbers and scales, on pages of every size that has its own kernel, and a
model of several layers on such a cache."""
import math

import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_cache8 import U, _random_cache, _slots, _write_both, bf16, f32
from tests.test_gpu_decoder import OPTS, _model
from tests.test_gpu_packed_model import PLAN, _dev, _walk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [bf16, f32], ids=str)
@pytest.mark.parametrize("B, Hkv, T, d, block, held, counts", [
    (2, 2, 70, 128, 32, (5, 0), (70, 50)),     # pages of 4096 values: eight pieces a lane of one wave
    (1, 2, 40, 256, 16, (3,), (40,)),
    (2, 1, 130, 64, 64, (60, 0), (130, 129)),
    (1, 2, 30, 136, 16, (15,), (30,)),         # just past 2048
    (1, 2, 150, 100, 64, (10,), (150,)),       # by element, four waves a page
    (2, 1, 200, 33, 128, (0, 127), (200, 130)),
    (1, 1, 90, 257, 40, (39,), (90,)),
    (1, 2, 40, 100, 40, (1,), (40,)),          # by element, one wave: more than it keeps
    (1, 1, 70, 256, 128, (5,), (70,)),         # past what four waves keep
])
def test_write_pages_of_every_size(B, Hkv, T, d, block, held, counts, dtype, code):
    announce("cache8 write, pages", T=T, d=d, block=block, dtype=dtype, code=code)
    g = torch.Generator().manual_seed(B + T + d)
    slots, blocks = _slots(B, T, block, held, counts, g)
    caches = [_random_cache(blocks, Hkv, block, d, code, g) for _ in range(2)]
    x = [(torch.randn(B, Hkv, T, d, generator=g) * torch.exp2(torch.randint(-6, 14, (B, Hkv, T, 1), generator=g).float()))
         .to(dtype) for _ in range(2)]
    _write_both(x, slots, caches, code, dtype)


class _Watched:
    """A cache that holds every written key and value a second time as it was, and looks at what comes back: what is read
    is off by the numbers' rounding alone, and attention is that over the values that are read."""

    def __init__(self, cache):
        self.cache = cache
        self.own = [[torch.zeros(x.shape, device="cuda") for x in xs] for xs in (cache.k, cache.v)]

    def __getattr__(self, name):
        return getattr(self.cache, name)

    def write(self, layer, k, v, slots):
        from edifice_amd import fused_scan as fs
        self.cache.write(layer, k, v, slots)
        fs.paged_cache_write(k, v, slots, self.own[0][layer], self.own[1][layer])

    def read(self, layer, offsets, total, dtype):
        from edifice_amd import fused_scan as fs
        got = self.cache.read(layer, offsets, total, dtype)
        want = fs.paged_cache_read(self.own[0][layer], self.own[1][layer], self.table, offsets, total)
        for x, y, scale in zip(got, want, (self.k_scale[layer], self.v_scale[layer])):
            # int8: half a step of the page's scale, and half of that for each time it doubled; e4m3: half a step of three
            # bits below the leading one, and the same series of the least step
            step = scale.max()
            bound = step if self.k[0].dtype == torch.int8 else y.abs() * 2.0 ** -4 + step * 2.0 ** -9
            assert bool(((x - y).abs() <= bound * (1 + 2.0 ** -20)).all())
            assert not total or bool(x.any())
        return got

    def attend(self, layer, q, window=0, sinks=0):
        got = self.cache.attend(layer, q, window, sinks)
        lengths = self.lengths.tolist()
        off = _dev(lengths)
        k, v = self.read(layer, off, sum(lengths), f32)
        for r, n in enumerate(lengths):
            if n:
                a = sum(lengths[:r])
                kr, vr = (t[:, a:a + n].repeat_interleave(q.shape[1] // k.shape[0], 0).double() for t in (k, v))
                s = (kr * q[r].reshape(q.shape[1], 1, -1).double()).sum(-1) * q.shape[-1] ** -0.5
                j = torch.arange(n, device="cuda")
                if window:
                    s = s.masked_fill((n - 1 - j >= window) & (j >= sinks), -math.inf)
                w = torch.softmax(s, -1)[..., None]
                want, size = (w * vr).sum(1), (w * vr.abs()).sum(1)
                # P times the scale in two float16 parts, 256 units of the float32 sums, the result's rounding
                tol = (2.0 ** -22 + 256 * U) * size + U * want.abs()
                assert bool(((got[r].reshape(want.shape) - want).abs() <= tol).all())
        return got


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("opts", [OPTS, {}], ids=str)
def test_layers_of_a_model_each_with_its_pages(code, opts):
    """Several layers on an 8-bit cache: each reads its own pages in units of its own scales, whatever the turns."""
    announce("8-bit layers", code=code, opts=opts)
    m = _model(f32, **opts)
    assert len(m.blocks) > 1
    g = torch.Generator().manual_seed(12)
    texts = [torch.randn(sum(n[r] for _, n in PLAN), 48, generator=g).cuda() for r in range(3)]
    plain = m.paged_cache(3, 200, block_size=16, dtype=code)
    cache = _Watched(m.paged_cache(3, 200, block_size=16, dtype=code))
    got, at = _walk(m, cache, texts, PLAN)
    again, _ = _walk(m, plain, texts, PLAN)
    assert cache.lengths.tolist() == at and all(torch.equal(a, b) for a, b in zip(got, again))
    scales = [*cache.k_scale, *cache.v_scale]
    assert not any(torch.equal(a, b) for i, a in enumerate(scales) for b in scales[:i])
