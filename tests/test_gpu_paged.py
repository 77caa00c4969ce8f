"""GPU parity: block tables and slots, the write into the pages, and attention over them.

Tolerances of the attention, per element: h (half a step of the type) for P and for the result, 256 units of 2^-24
for the float32 sums, of the sum of the terms' sizes (oracle/decoder.py returns it).  The others are exact."""
import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
H = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
bf16, f32 = torch.bfloat16, torch.float32

EXTEND = [
    # (R, width, block, tokens, free, longest)
    (1, 1, 16, 1, 4, 16),
    (5, 8, 4, 3, 60, 32),
    (70, 6, 16, 1, 80, 96),      # decode step
    (3, 40, 16, 600, 200, 640),  # prompts over several workgroups
    (9, 4, 8, 5, 6, 40),         # the list runs out, lengths past the table
    (2000, 3, 2, 1, 3000, 8),    # requests over several workgroups
    (4, 9, 7, 2, 40, 60),        # block no power of two, more growth than tokens asked for
]


@pytest.mark.parametrize("case", EXTEND, ids=str)
def test_paged_extend(case):
    from edifice_amd import fused_scan as fs
    R, width, block, tokens, free, longest = case
    announce("paged_extend", case=case)
    g = torch.Generator().manual_seed(R)
    old = torch.randint(-2, longest + 1, (R,), generator=g)
    new = old + torch.randint(-2, max(tokens, 3 * block) + 1, (R,), generator=g)
    table = torch.full((R, width), -1, dtype=torch.int64)
    ids = torch.randperm(4 * R * width + free, generator=g)
    at = 0
    for r in range(R):
        n = min(-(-max(int(old[r]), 0) // block), width)
        table[r, :n] = ids[at:at + n]
        at += n
    fr = ids[at:at + free]
    i32 = lambda t: t.to(torch.int32).cuda()  # noqa: E731
    td = i32(table)
    slots, pos, used = fs.paged_extend(td, i32(old), i32(new), i32(fr), block, tokens)
    want = od.paged_extend(table.tolist(), old.tolist(), new.tolist(), fr.tolist(), block, tokens)
    assert td.tolist() == want[0]
    assert slots.tolist() == want[1]
    assert pos.tolist() == want[2]
    assert used.tolist() == [want[3]]


@pytest.mark.parametrize("taken", [-3, 2, 5, 2**31 - 1])
def test_paged_extend_after_a_count(taken):
    """Entries gone before the call: a negative count is none; past the list, whatever the sum, no page is given."""
    from edifice_amd import fused_scan as fs
    announce("paged_extend taken", taken=taken)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    free = [7, 3, 9, 1, 4]
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    slots, pos, used = fs.paged_extend(table, i32([0, 0, 0]), i32([1, 5, 3]), i32(free), 4, 5, i32([taken]))
    at = max(taken, 0)
    pages = [free[at + i] if at + i < len(free) else -1 for i in range(4)]
    want = [[pages[0], -1], [pages[1], pages[2]], [pages[3], -1]]
    assert table.tolist() == want
    assert used.tolist() == [min(at + 4, 2**31 - 1)]
    for r, n in enumerate([1, 5, 3]):
        assert pos[r].tolist() == [t if t < n else -1 for t in range(5)]
        assert slots[r].tolist() == [want[r][t // 4] * 4 + t % 4 if t < n and want[r][t // 4] >= 0 else -1
                                     for t in range(5)]


@pytest.mark.parametrize("case", [(2, 3, 5, 64, 8, bf16), (1, 1, 1, 128, 16, f32), (3, 2, 70, 7, 4, bf16),
                                  (2, 2, 9, 5, 3, f32)], ids=str)
def test_paged_cache_write(case):
    """Each token's rows land in their slot and nothing else changes: slots of -1 and past the cache are left out."""
    from edifice_amd import fused_scan as fs
    B, Hkv, T, d, block, dtype = case
    announce("paged_cache_write", case=case)
    g = torch.Generator().manual_seed(1)
    blocks = B * T // block + 4
    k, v = (torch.randn(B, Hkv, T, d, generator=g).to(dtype) for _ in range(2))
    kc, vc = (torch.randn(blocks, Hkv, block, d, generator=g).to(dtype) for _ in range(2))
    slots = torch.randperm(blocks * block, generator=g)[:B * T].view(B, T).to(torch.int32)
    if T > 1:
        slots[0, 0], slots[-1, 1], slots[-1, 2] = -1, blocks * block, -2 ** 31
    kd, vd = kc.cuda(), vc.cuda()
    fs.paged_cache_write(k.cuda(), v.cuda(), slots.cuda(), kd, vd)
    for b in range(B):
        for t in range(T):
            s = int(slots[b, t])
            if 0 <= s < blocks * block:
                kc[s // block, :, s % block], vc[s // block, :, s % block] = k[b, :, t], v[b, :, t]
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


PAGED = [
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
]


def _pool(lengths, Hkv, d, block, dtype, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    width = max(1, -(-max(lengths) // block)) + 2
    total = sum(-(-n // block) for n in lengths) + spare
    ids = torch.randperm(total, generator=g)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        m = -(-n // block)
        table[b, :m] = ids[at:at + m].to(torch.int32)
        at += m
    kc, vc = (torch.randn(total, Hkv, block, d, generator=g).to(dtype) for _ in range(2))
    return kc, vc, table, torch.tensor(lengths, dtype=torch.int32), g


def _check(got, q, kc, vc, table, lengths, window, sinks, dtype):
    want, mag = od.paged_attention(q.double(), kc.double(), vc.double(), table, lengths, window, sinks)
    h = H[dtype] if dtype == bf16 else 0.0
    tol = (h + 256 * U) * mag + max(h, U) * want.abs()
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol).max()):.3e}"


@pytest.mark.parametrize("case", PAGED, ids=str)
def test_paged_attention(case):
    from edifice_amd import fused_scan as fs
    lengths, Hq, Hkv, d, block, window, sinks, dtype = case
    announce("paged_attention", case=case)
    kc, vc, table, n, g = _pool(lengths, Hkv, d, block, dtype)
    q = torch.randn(len(lengths), Hq, d, generator=g).to(dtype)
    # what lies behind a request's end, and in pages that nobody holds, is not read into the result
    used = torch.zeros(kc.shape[0], block, dtype=torch.bool)
    for b, m in enumerate(lengths):
        for j in range(m):
            used[table[b, j // block], j % block] = True
    for c in (kc, vc):
        c.transpose(1, 2)[~used] = float("nan")
    dev = [t.cuda() for t in (q, kc, vc, table, n)]
    got = fs.paged_attention(*dev, window=window, sinks=sinks)
    clean = [torch.nan_to_num(c) for c in (kc, vc)]
    _check(got, q, *clean, table, n, window, sinks, dtype)
    assert torch.equal(fs.paged_attention(dev[0][:, :, None], *dev[1:], window=window, sinks=sinks)[:, :, 0], got)


def test_a_window_without_end():
    """A window and sinks past any int see every key, as no window does."""
    from edifice_amd import fused_scan as fs
    announce("paged_window_without_end")
    kc, vc, table, n, g = _pool([70, 5], 2, 64, 16, f32)
    dev = [t.cuda() for t in (torch.randn(2, 4, 64, generator=g), kc, vc, table, n)]
    want = fs.paged_attention(*dev)
    for window, sinks in ((2**63 - 1, 0), (2**32 + 3, 0), (1, 2**32 + 3)):
        _check(fs.paged_attention(*dev, window=window, sinks=sinks), dev[0].cpu(), kc, vc, table, n, 0, 0, f32)
    assert torch.equal(fs.paged_attention(*dev, window=0, sinks=2**32 + 3), want)


@pytest.mark.parametrize("dtype", [bf16, f32], ids=str)
def test_pages_one_element_off(dtype):
    """Caches and queries whose rows are off 16 bytes: the write and the attention by elements."""
    from edifice_amd import fused_scan as fs
    announce("paged_off", dtype=dtype)

    def off(t):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)
    kc, vc, table, n, g = _pool([150, 33], 2, 64, 16, dtype)
    q = torch.randn(2, 6, 64, generator=g).to(dtype)
    k, v = (torch.randn(2, 2, 1, 64, generator=g).to(dtype) for _ in range(2))
    kd, vd, qd = off(kc), off(vc), off(q)
    slots = torch.stack([table[b, (n[b] - 1) // 16] * 16 + (n[b] - 1) % 16 for b in range(2)])[:, None]
    fs.paged_cache_write(off(k), off(v), slots.to(torch.int32).cuda(), kd, vd)
    for b in range(2):
        s = int(slots[b])
        kc[s // 16, :, s % 16], vc[s // 16, :, s % 16] = k[b, :, 0], v[b, :, 0]
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)
    _check(fs.paged_attention(qd, kd, vd, table.cuda(), n.cuda()), q, kc, vc, table, n, 0, 0, dtype)


def test_bad_pages_and_lengths():
    """Page numbers outside the cache hold no keys; a length past the table counts to the table's end, a negative
    one as none.  (The kernel checks each number against the cache before it forms an address.)"""
    from edifice_amd import fused_scan as fs
    announce("paged_bad_pages")
    kc, vc, table, n, g = _pool((40, 64, 10), 2, 64, 8, f32)
    table[0, 1], table[0, 3], table[1, :], table[2, 0] = -1, kc.shape[0], 2 ** 31 - 1, -2 ** 31
    table[2, 1:] = 0
    n = torch.tensor([40, 64, 2 ** 31 - 1], dtype=torch.int32)
    q = torch.randn(3, 2, 64, generator=g)
    got = fs.paged_attention(*(t.cuda() for t in (q, kc, vc, table, n)))
    _check(got, q, kc, vc, table, n, 0, 0, f32)
    assert not got[1].any()  # no key at all
    n[2] = -5
    assert not fs.paged_attention(*(t.cuda() for t in (q, kc, vc, table, n)))[2].any()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements (4.3 GB each): pages at its far end."""
    from edifice_amd import fused_scan as fs
    announce("paged_far_pages")
    blocks, Hkv, block, d = (1 << 31) // (16 * 128) // 2 + 1000, 2, 16, 128
    kc, vc = (torch.zeros(blocks, Hkv, block, d, dtype=bf16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, Hkv, 40, d, generator=g).to(bf16) for _ in range(2))
    table = torch.tensor([[blocks - 1, blocks - 7, 3]], dtype=torch.int32)
    t = torch.arange(40)
    slots = (table[0, t // 16].long() * 16 + t % 16).to(torch.int32)[None]
    fs.paged_cache_write(k.cuda(), v.cuda(), slots.cuda(), kc, vc)
    assert torch.equal(kc[blocks - 1].cpu(), k[0, :, :16]) and torch.equal(vc[blocks - 7].cpu(), v[0, :, 16:32])
    q = torch.randn(1, 4, d, generator=g).to(bf16)
    got = fs.paged_attention(q.cuda(), kc, vc, table.cuda(), torch.tensor([40], dtype=torch.int32, device="cuda"))
    pages = lambda u: torch.cat([u, u.new_zeros(1, Hkv, 8, d)], 2).view(Hkv, 3, 16, d).transpose(0, 1)  # noqa: E731
    _check(got, q, pages(k), pages(v), torch.tensor([[0, 1, 2]]), torch.tensor([40]), 0, 0, bf16)


def test_captured_decode_replays_with_new_lengths():
    """Extend, write and attend in one graph; lengths and tokens change between the replays."""
    from edifice_amd import fused_scan as fs
    announce("paged_graph")
    B, Hq, Hkv, d, block, width = 3, 4, 2, 64, 4, 8
    g = torch.Generator().manual_seed(4)
    kc, vc = (torch.zeros(B * width, Hkv, block, d, dtype=bf16, device="cuda") for _ in range(2))
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(B * width, generator=g).to(torch.int32)
    old, new = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    fd = free.cuda()
    q, k, v = (torch.zeros(B, h, 1, d, dtype=bf16, device="cuda") for h in (Hq, Hkv, Hkv))

    def step():
        slots, _, used = fs.paged_extend(table, old, new, fd, block, 1)
        fs.paged_cache_write(k, v, slots, kc, vc)
        return fs.paged_attention(q, kc, vc, table, new), used

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, used = step()
    keys, vals, at = [[] for _ in range(B)], [[] for _ in range(B)], 0
    for i in range(11):
        grow = torch.tensor([1, int(i % 2 == 0), int(i > 3)], dtype=torch.int32)
        for t, h in ((q, Hq), (k, Hkv), (v, Hkv)):
            t.copy_(torch.randn(B, h, 1, d, generator=g).to(bf16))
        old.copy_(new)
        new.copy_(old + grow.cuda())
        fd.copy_(torch.cat([free[at:], free[:at]]))
        graph.replay()
        at += int(used)
        for b in range(B):
            if grow[b]:
                keys[b].append(k[b, :, 0].cpu())
                vals[b].append(v[b, :, 0].cpu())
            if keys[b]:
                kk, vv = (torch.stack(s, 1)[None] for s in (keys[b], vals[b]))  # one page of all tokens
                _check(out[b:b + 1, :, 0], q[b:b + 1, :, 0].cpu(), kk, vv, torch.zeros(1, 1, dtype=torch.int32),
                       torch.tensor([len(keys[b])]), 0, 0, bf16)
            else:
                assert not out[b].any()
