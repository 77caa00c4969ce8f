"""GPU parity of the 8-bit paged cache: the write (numbers and scales exactly), reading back (exactly), and the attention
of one token over it.

Tolerance of the attention, per element: P in its bf16 parts (2^-16 in bf16, 2^-24 in float32) and 256 units of 2^-24 for
the float32 sums, of the sum of the terms' sizes (oracle/decoder.py returns it), and half a step of the type of the result."""
import math

import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
bf16, f32 = torch.bfloat16, torch.float32
KIND = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _random_cache(blocks, Hkv, block, d, code, g):
    """Numbers of the kind in every place, as float64, and scales of 2^-4 .. 2^4 times something."""
    if code == "int8":
        c = torch.randint(-127, 128, (blocks, Hkv, block, d), generator=g).double()
    else:
        c = od.round_code((torch.randn(blocks, Hkv, block, d, generator=g) * 40).double().clamp(-448, 448), code)
    s = torch.exp2(torch.randint(-4, 5, (blocks, Hkv), generator=g).float())
    return c, s * (1 + torch.rand(blocks, Hkv, generator=g)) if code == "int8" else s


def _slots(B, T, block, held, counts, g, spare=2):
    """Slots of tokens held[b] .. of each row, in pages of random order; -1 past counts[b]."""
    width = -(-(max(held) + T) // block)
    ids = torch.randperm(B * width + spare, generator=g).tolist()
    return [[ids[b * width + (held[b] + t) // block] * block + (held[b] + t) % block if t < counts[b] else -1
             for t in range(T)] for b in range(B)], B * width + spare


def _to_gpu(c, s, code):
    return c.float().to(KIND[code]).cuda(), s.float().cuda()


def _same(got_c, got_s, c, s):
    assert torch.equal(got_s.cpu().nan_to_num(-1.0), s.float().nan_to_num(-1.0))
    assert torch.equal(got_c.cpu().float().double(), c)


def _write_both(x, slots, caches, code, dtype):
    """The operator and the oracle on the same keys and values; returns what the operator left."""
    from edifice_amd import fused_scan as fs
    (kc, ks), (vc, vs) = caches
    (kd, ksd), (vd, vsd) = _to_gpu(kc, ks, code), _to_gpu(vc, vs, code)
    fs.paged_cache_write(x[0].cuda(), x[1].cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), kd, vd, ksd, vsd)
    od.paged_cache_write8(x[0].double(), slots, kc, ks, code)
    od.paged_cache_write8(x[1].double(), slots, vc, vs, code)
    _same(kd, ksd, kc, ks)
    _same(vd, vsd, vc, vs)
    return kd, vd, ksd, vsd


WRITE = [
    # (B, Hkv, T, d, block, held, counts, dtype)
    (1, 1, 1, 64, 16, (0,), (1,), bf16),               # one token begins a page
    (3, 2, 1, 128, 16, (5, 16, 31), (1, 1, 1), bf16),  # a decode step: inside, at the start and at the end of a page
    (2, 2, 40, 64, 16, (0, 3), (40, 33), bf16),        # prompts into fresh pages, one onto a page that holds some
    (1, 3, 70, 128, 16, (7,), (70,), f32),             # a page's tokens across the 16 that a wave looks at
    (2, 1, 150, 40, 128, (100, 0), (150, 130), bf16),  # pages of 128: four waves a page, across 64 tokens
    (1, 2, 300, 256, 128, (60,), (300,), f32),
    (2, 2, 9, 7, 4, (2, 0), (9, 5), bf16),             # rows off 16 bytes
    (1, 1, 5, 33, 3, (1,), (5,), f32),                 # block no power of two
    (2, 1, 1, 512, 64, (63, 70), (1, 1), bf16),
    (4, 2, 3, 64, 1, (0, 1, 2, 5), (3, 0, 1, 2), f32),  # pages of one token, a row without tokens
    (1, 1, 200, 16, 100, (0,), (200,), bf16),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", WRITE, ids=str)
def test_write(case, code):
    B, Hkv, T, d, block, held, counts, dtype = case
    announce("cache8 write", case=case, code=code)
    g = torch.Generator().manual_seed(B + T)
    slots, blocks = _slots(B, T, block, held, counts, g)
    caches = [_random_cache(blocks, Hkv, block, d, code, g) for _ in range(2)]
    # from values far below the pages' scales to values that double them several times
    x = [(torch.randn(B, Hkv, T, d, generator=g) * torch.exp2(torch.randint(-6, 14, (B, Hkv, T, 1), generator=g).float()))
         .to(dtype) for _ in range(2)]
    _write_both(x, slots, caches, code, dtype)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_token_by_token(code):
    """A text written one token at a time, ever larger ones among them: exactly the definition's numbers after each, and
    at the end no value further off than a step of its page's scale (int8), or than its own rounding and the least step (e4m3)."""
    from edifice_amd import fused_scan as fs
    announce("cache8 decode", code=code)
    g = torch.Generator().manual_seed(3)
    Hkv, d, block, T = 2, 64, 8, 30
    zero = lambda: [torch.zeros(5, Hkv, block, d, dtype=torch.float64), torch.zeros(5, Hkv, dtype=torch.float64)]  # noqa: E731
    kc, vc = zero(), zero()
    kd, ksd = _to_gpu(*kc, code)
    vd, vsd = _to_gpu(*vc, code)
    x = [torch.randn(1, Hkv, T, d, generator=g) * torch.exp2(0.3 * torch.arange(T, dtype=f32))[:, None] for _ in range(2)]
    pages = [3, 0, 4, 1]
    for t in range(T):
        slots = [[pages[t // block] * block + t % block]]
        k, v = (u[:, :, t:t + 1].contiguous() for u in x)
        fs.paged_cache_write(k.cuda(), v.cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), kd, vd, ksd, vsd)
        od.paged_cache_write8(k.double(), slots, *kc, code)
        od.paged_cache_write8(v.double(), slots, *vc, code)
        _same(kd, ksd, *kc)
        _same(vd, vsd, *vc)
    table = torch.tensor([pages], dtype=torch.int32).cuda()
    k, v = fs.paged_cache_read(kd, vd, table, torch.tensor([0, T], dtype=torch.int32).cuda(), T, ksd, vsd, dtype=f32)
    for got, want, scale in ((k, x[0][0], ksd), (v, x[1][0], vsd)):
        step = scale.cpu()[[pages[t // block] for t in range(T)]].T[:, :, None]
        off = (got.cpu() - want).abs()
        # int8: half a step, and half of that for each halving: 1/2 + 1/4 + ... of the last scale.  e4m3: half a step of three
        # bits below the value's leading one, 2^-4 of it, and the same series of the fixed step 2^-9 once it is below 2^-6
        bound = step if code == "int8" else want.abs() * 2.0 ** -4 + step * 2.0 ** -9
        assert bool((off <= bound * (1 + 2.0 ** -20)).all()), float((off / bound).max())


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_zeros_tiny_large_and_not_finite(code):
    announce("cache8 write, special values", code=code)
    g = torch.Generator().manual_seed(4)
    B, Hkv, T, d, block = 8, 1, 4, 32, 4
    x = [torch.randn(B, Hkv, T, d, generator=g) for _ in range(2)]
    for u in x:
        u[0] = 0.0                       # a page of zeros
        u[1] *= 2.0 ** -140              # below the least scale
        u[2] *= 2.0 ** 120
        u[3, 0, 1, 5] = math.nan
        u[4, 0, 0, 0] = -math.inf
        u[5, 0, 2, 3] = -0.0
        u[6] = 448.0 * 2.0 ** -3         # e4m3: exactly the largest number of a scale
        u[7] = 449.0 * 2.0 ** -3         # and past it
    slots, blocks = _slots(B, T, block, (0,) * B, (T,) * B, g)
    caches = [_random_cache(blocks, Hkv, block, d, code, g) for _ in range(2)]
    _, _, ks, _ = _write_both(x, slots, caches, code, f32)
    pages = [row[0] // block for row in slots]
    assert ks[pages[0], 0] == 0 and torch.isnan(ks[pages[3], 0]) and torch.isnan(ks[pages[4], 0])
    # the same pages go on behind their first two tokens: zeros grow, what is not finite stays so
    later = [[-1, -1] + row[2:] for row in slots]
    y = [torch.randn(B, Hkv, T, d, generator=g) for _ in range(2)]
    _write_both(y, later, caches, code, f32)
    # and start anew
    _, _, ks, _ = _write_both(y, slots, caches, code, f32)
    assert bool(torch.isfinite(ks[pages]).all())


def test_write_leaves_out_slots_outside_the_cache():
    announce("cache8 write, slots outside")
    g = torch.Generator().manual_seed(5)
    slots = [[0, 1, 2, 3, -1, 40, 2 ** 31 - 1, -2 ** 31, 12, 13]]
    caches = [_random_cache(5, 2, 8, 16, "int8", g) for _ in range(2)]  # 40 slots
    x = [torch.randn(1, 2, 10, 16, generator=g) for _ in range(2)]
    _write_both(x, slots, caches, "int8", f32)


READ = [
    # (lengths, Hkv, d, block, spare rows behind)
    ((1,), 1, 64, 16, 0),
    ((0, 5, 33, 0), 2, 128, 16, 3),
    ((130, 1, 64), 3, 80, 32, 0),
    ((9, 4), 2, 7, 4, 2),
    ((70, 200), 1, 256, 128, 65),
    ((3, 0, 0, 2), 2, 33, 1, 0),
]


@pytest.mark.parametrize("kind", ["int8", "e4m3", "f32", "bf16"])
@pytest.mark.parametrize("case", READ, ids=str)
def test_read(case, kind):
    from edifice_amd import fused_scan as fs
    lengths, Hkv, d, block, behind = case
    announce("cache read", case=case, kind=kind)
    g = torch.Generator().manual_seed(len(lengths))
    width = max(1, -(-max(lengths) // block)) + 1
    blocks = len(lengths) * width + 1
    table = torch.randperm(blocks, generator=g)[:len(lengths) * width].view(-1, width).to(torch.int32)
    if max(lengths) > block:  # a page that was not found, and one outside the cache
        table[lengths.index(max(lengths)), 0] = -1
        table[lengths.index(max(lengths)), 1] = blocks
    offsets = [0] + torch.tensor(lengths).cumsum(0).tolist()
    total = offsets[-1] + behind
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    if kind in KIND:
        caches = [_random_cache(blocks, Hkv, block, d, kind, g) for _ in range(2)]
        (kd, ks), (vd, vs) = (_to_gpu(*c, kind) for c in caches)
        values = [c.float() * s.float()[:, :, None, None] for c, s in caches]
        outs = [(dt, fs.paged_cache_read(kd, vd, table.cuda(), off, total, ks, vs, dtype=dt)) for dt in (f32, bf16)]
        outs.append((bf16, fs.paged_cache_read(kd, vd, table.cuda(), off, total, ks, vs)))
    else:
        dt = f32 if kind == "f32" else bf16
        values = [torch.randn(blocks, Hkv, block, d, generator=g).to(dt) for _ in range(2)]
        outs = [(dt, fs.paged_cache_read(values[0].cuda(), values[1].cuda(), table.cuda(), off, total))]
    for dt, got in outs:
        for x, y in zip(got, values):
            assert x.dtype == dt
            assert torch.equal(x.cpu(), od.paged_cache_read(y, table, offsets, total).to(dt))


def test_read_offsets_out_of_order_stay_in_bounds():
    """Offsets that do not ascend give some rows, none from outside the cache: every row is one of its or zeros."""
    from edifice_amd import fused_scan as fs
    announce("cache read, offsets out of order")
    kc = torch.ones(4, 1, 2, 8).cuda()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    for offsets in ([0, 9, 4], [-5, 3, 2], [3, 3, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, 0]):
        k, _ = fs.paged_cache_read(kc, kc, table, torch.tensor(offsets, dtype=torch.int32).cuda(), 6)
        assert bool(((k == 0) | (k == 1)).all())


ATTEND = [
    # (lengths, Hq, Hkv, d, block, window, sinks, dtype)
    ((1,), 1, 1, 64, 16, 0, 0, bf16),
    ((0, 5, 33), 4, 2, 128, 16, 0, 0, bf16),             # an empty place
    ((700, 129, 128, 127), 8, 1, 64, 32, 0, 0, bf16),    # pages that end inside a tile
    ((1000, 3, 260), 6, 2, 128, 64, 100, 4, bf16),       # window and sinks
    ((300, 50), 40, 2, 128, 16, 0, 0, bf16),             # 20 query heads a key head: two query tiles
    ((90, 41), 4, 4, 80, 8, 33, 0, bf16),
    ((90, 41), 3, 1, 7, 4, 0, 0, bf16),                  # rows off 16 bytes
    ((130, 77), 4, 2, 256, 16, 0, 0, bf16),
    ((130, 77), 2, 1, 250, 3, 0, 0, bf16),               # block no power of two
    ((500, 0, 64), 4, 2, 64, 16, 0, 0, f32),
    ((210, 31), 7, 1, 128, 32, 64, 20, f32),
    ((95, 96, 97), 2, 2, 256, 1, 0, 0, f32),             # pages of one token
    ((61, 9), 2, 1, 33, 5, 10, 3, f32),
    ((5000,), 2, 1, 128, 16, 0, 0, bf16),                # split over the length
    ((4000, 1), 2, 2, 48, 16, 0, 0, f32),
]


def _pool(lengths, Hkv, block, d, code, g, spare=3):
    width = max(1, -(-max(lengths) // block)) + 2
    total = sum(-(-n // block) for n in lengths) + spare
    ids = torch.randperm(total, generator=g)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        m = -(-n // block)
        table[b, :m] = ids[at:at + m].to(torch.int32)
        at += m
    caches = []
    for _ in range(2):
        x = torch.randn(total, Hkv, block, d, generator=g).double()
        c, s = torch.zeros_like(x), torch.zeros(total, Hkv, dtype=torch.float64)
        for p in range(total):
            for h in range(Hkv):
                s[p, h] = od.least_scale(float(x[p, h].abs().max()), code)
        c = od.round_code(x / s[:, :, None, None], code)
        caches.append((c, s))
    return caches, table, torch.tensor(lengths, dtype=torch.int32)


def _expect(got, q, caches, table, lengths, window, sinks, dtype):
    values = [c * s.float().double()[:, :, None, None] for c, s in caches]
    want, mag = od.paged_attention(q.double(), *values, table, lengths, window, sinks)
    p, h = (2.0 ** -16, 2.0 ** -8) if dtype == bf16 else (U, U)
    tol = (p + 256 * U) * mag + h * want.abs()
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol).max()):.3e}"


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attention(case, code):
    from edifice_amd import fused_scan as fs
    lengths, Hq, Hkv, d, block, window, sinks, dtype = case
    announce("paged_attention8", case=case, code=code)
    g = torch.Generator().manual_seed(1)
    caches, table, n = _pool(lengths, Hkv, block, d, code, g)
    q = torch.randn(len(lengths), Hq, d, generator=g).to(dtype)
    (kd, ks), (vd, vs) = (_to_gpu(*c, code) for c in caches)
    # what lies behind a request's end, and in pages that nobody holds, is not read into the result
    held = torch.zeros(kd.shape[0], block, dtype=torch.bool)
    for b, m in enumerate(lengths):
        for j in range(m):
            held[int(table[b, j // block]), j % block] = True
    worst = -128 if code == "int8" else 0x7F  # e4m3's NaN
    for c, s in ((kd, ks), (vd, vs)):
        c.view(torch.int8).permute(0, 2, 1, 3)[~held.cuda()] = worst
        s[~held.any(1).cuda()] = math.nan
    _expect(fs.paged_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), window=window, sinks=sinks, k_scale=ks,
                               v_scale=vs), q, caches, table, n, window, sinks, dtype)


def _ragged(n, top):
    return tuple((i * 7919 + 13) % (top + 1) for i in range(n - 1)) + (top,)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("case", [
    (_ragged(3, 766), 8, 4, 64, 16, 0, 0, f32),      # whole requests, a few and many of them
    (_ragged(270, 120), 1, 1, 64, 16, 0, 0, bf16),
    (_ragged(130, 1500), 4, 2, 128, 16, 0, 0, bf16),
    (_ragged(100, 900), 3, 3, 48, 8, 200, 3, bf16),
    (_ragged(90, 700), 3, 3, 33, 5, 0, 0, f32),
    (_ragged(6, 1100), 4, 2, 128, 16, 0, 0, f32),    # cut, few and many
    (_ragged(90, 2300), 3, 3, 64, 64, 0, 0, bf16),
    (_ragged(3, 769), 2, 1, 256, 16, 700, 60, bf16),
    (_ragged(5, 2000), 6, 2, 128, 64, 800, 20, bf16),
    (_ragged(3, 1500), 40, 2, 64, 16, 0, 0, bf16),   # two query tiles
    (_ragged(3, 1300), 4, 4, 80, 8, 1000, 0, bf16),
    (_ragged(3, 900), 3, 1, 33, 5, 0, 0, bf16),      # rows by element
    (_ragged(3, 1000), 7, 1, 100, 32, 770, 3, f32),
    (_ragged(2, 800), 2, 2, 7, 1, 0, 0, f32),
], ids=lambda c: f"{len(c[0])}to{max(c[0])}-" + "-".join(str(x) for x in c[1:]))
def test_attention_of_whole_and_cut_requests(case, code):
    test_attention(case, code)


def test_attention_without_some_pages():
    from edifice_amd import fused_scan as fs
    announce("paged_attention8, pages missing")
    g = torch.Generator().manual_seed(2)
    caches, table, n = _pool((100, 40, 16), 2, 16, 64, "int8", g)
    table[0, 2], table[1, 0], table[2, 0] = -1, caches[0][0].shape[0], -5
    q = torch.randn(3, 4, 64, generator=g)
    (kd, ks), (vd, vs) = (_to_gpu(*c, "int8") for c in caches)
    _expect(fs.paged_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), k_scale=ks, v_scale=vs), q, caches, table, n, 0,
            0, f32)


def test_attention_scales_far_apart():
    """Pages whose scales are 2^-90 and 2^20 next to one another: no product of a scale alone leaves float32's range."""
    from edifice_amd import fused_scan as fs
    announce("paged_attention8, scales far apart")
    g = torch.Generator().manual_seed(6)
    caches, table, n = _pool((64,), 1, 16, 64, "e4m3", g)
    (kc, ks), (vc, vs) = caches
    ks[table[0, 1].long()] *= 2.0 ** -90
    vs[table[0, 2].long()] *= 2.0 ** -90
    vs[table[0, 3].long()] *= 2.0 ** 20
    q = torch.randn(1, 2, 64, generator=g)
    (kd, ksd), (vd, vsd) = (_to_gpu(*c, "e4m3") for c in caches)
    _expect(fs.paged_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), k_scale=ksd, v_scale=vsd), q, caches, table, n, 0,
            0, f32)


def test_pages_of_zeros_before_tiny_ones():
    """Pages whose scale is 0 (all zeros) do not set what later, tiny ones are held against."""
    from edifice_amd import fused_scan as fs
    announce("paged_attention8, zeros before tiny values")
    for code, dtype in (("int8", f32), ("e4m3", bf16)):
        g = torch.Generator().manual_seed(10)
        caches, table, n = _pool((300,), 1, 16, 64, code, g)
        (kc, ks), (vc, vs) = caches
        vs *= 2.0 ** -80
        vs[table[0, :8].long()] = 0.0
        q = torch.randn(1, 2, 64, generator=g).to(dtype)
        (kd, ksd), (vd, vsd) = (_to_gpu(*c, code) for c in caches)
        got = fs.paged_attention(q.cuda(), kd, vd, table.cuda(), n.cuda(), k_scale=ksd, v_scale=vsd)
        assert bool(got.any())
        _expect(got, q, caches, table, n, 0, 0, dtype)


def test_page_that_is_not_finite_reaches_who_sees_it():
    from edifice_amd import fused_scan as fs
    announce("paged_attention8, a page of NaN")
    g = torch.Generator().manual_seed(7)
    caches, table, n = _pool((40, 40), 1, 8, 32, "int8", g)
    (kd, ks), (vd, vs) = (_to_gpu(*c, "int8") for c in caches)
    q = torch.randn(2, 1, 32, generator=g).cuda()
    ks[table[0, 1].long(), 0] = math.nan
    call = lambda w: fs.paged_attention(q, kd, vd, table.cuda(), n.cuda(), window=w, k_scale=ks, v_scale=vs)  # noqa: E731
    got = call(0)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    assert bool(torch.isfinite(call(20)).all())  # the window begins behind it
    ks[table[0, 1].long(), 0], vs[table[0, 1].long(), 0] = 1.0, math.nan
    assert bool(torch.isnan(call(0)[0]).all()) and bool(torch.isfinite(call(20)).all())


def test_past_two_to_the_31_bytes():
    """The last pages of a cache of more than 2^31 bytes: written, attended to and read back."""
    from edifice_amd import fused_scan as fs
    announce("cache8 past 2^31 bytes")
    Hkv, block, d, blocks = 4, 128, 256, 17000  # 2.2 GB
    g = torch.Generator().manual_seed(8)
    kd, vd = (torch.zeros(blocks, Hkv, block, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(blocks, Hkv, device="cuda") for _ in range(2))
    k, v = (torch.randn(1, Hkv, 200, d, generator=g) for _ in range(2))
    pages = [blocks - 1, blocks - 2]
    slots = torch.tensor([[pages[t // block] * block + t % block for t in range(200)]], dtype=torch.int32).cuda()
    fs.paged_cache_write(k.cuda(), v.cuda(), slots, kd, vd, ks, vs)
    small = [[torch.zeros(2, Hkv, block, d, dtype=torch.float64), torch.zeros(2, Hkv, dtype=torch.float64)] for _ in range(2)]
    near = [[(t // block) * block + t % block for t in range(200)]]
    for x, c in zip((k, v), small):
        od.paged_cache_write8(x.double(), near, *c, "int8")
    _same(kd[pages], ks[pages], *small[0])
    _same(vd[pages], vs[pages], *small[1])
    table, n = torch.tensor([pages], dtype=torch.int32).cuda(), torch.tensor([200], dtype=torch.int32)
    off = torch.tensor([0, 200], dtype=torch.int32).cuda()
    got = fs.paged_cache_read(kd, vd, table, off, 200, ks, vs, dtype=f32)
    for x, (c, s) in zip(got, small):
        values = c.float() * s.float()[:, :, None, None]
        assert torch.equal(x.cpu(), values.transpose(0, 1).reshape(Hkv, -1, d)[:, :200])
    q = torch.randn(1, 8, d, generator=g)
    _expect(fs.paged_attention(q.cuda(), kd, vd, table, n.cuda(), k_scale=ks, v_scale=vs), q, small,
            torch.tensor([[0, 1]], dtype=torch.int32), n, 0, 0, f32)


def test_captured_on_another_stream():
    """A decode step (write, attend, read back) captured and replayed after the inputs have changed."""
    from edifice_amd import fused_scan as fs
    announce("cache8 captured")
    g = torch.Generator().manual_seed(9)
    Hkv, d, block = 2, 64, 16
    caches, table, n = _pool((50, 20), Hkv, block, d, "e4m3", g)
    (kd, ks), (vd, vs) = (_to_gpu(*c, "e4m3") for c in caches)
    start = [t.clone() for t in (kd.view(torch.int8), vd.view(torch.int8), ks, vs)]
    table, n = table.cuda(), n.cuda()
    off = torch.tensor([0, 50, 70], dtype=torch.int32).cuda()
    q, k, v = torch.zeros(2, 4, d).cuda(), torch.zeros(2, Hkv, 1, d).cuda(), torch.zeros(2, Hkv, 1, d).cuda()
    slots = torch.stack([table[b, (n[b] - 1) // block] * block + (n[b] - 1) % block for b in range(2)])[:, None].contiguous()

    def step():
        fs.paged_cache_write(k, v, slots, kd, vd, ks, vs)
        o = fs.paged_attention(q, kd, vd, table, n, k_scale=ks, v_scale=vs)
        return (o, *fs.paged_cache_read(kd, vd, table, off, 70, ks, vs, dtype=f32))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g) * 2 ** i)
        again = lambda: [a.copy_(b) for a, b in zip((kd.view(torch.int8), vd.view(torch.int8), ks, vs), start)]  # noqa: E731
        again()
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        again()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_empty_calls():
    from edifice_amd import fused_scan as fs
    announce("cache8 empty")
    i32 = dict(dtype=torch.int32, device="cuda")
    kc, s = torch.zeros(2, 1, 4, 8, dtype=torch.int8, device="cuda"), torch.zeros(2, 1, device="cuda")
    fs.paged_cache_write(torch.zeros(0, 1, 3, 8).cuda(), torch.zeros(0, 1, 3, 8).cuda(), torch.zeros(0, 3, **i32), kc, kc, s, s)
    k, v = fs.paged_cache_read(kc, kc, torch.zeros(0, 2, **i32), torch.zeros(1, **i32), 3, s, s)
    assert k.shape == v.shape == (1, 3, 8) and not k.any() and not v.any()
    k, _ = fs.paged_cache_read(kc, kc, torch.zeros(1, 2, **i32), torch.zeros(2, **i32), 0, s, s)
    assert k.shape == (1, 0, 8)
    o = fs.paged_attention(torch.zeros(0, 2, 8).cuda(), kc, kc, torch.zeros(0, 2, **i32), torch.zeros(0, **i32), k_scale=s,
                           v_scale=s)
    assert o.shape == (0, 2, 8)
