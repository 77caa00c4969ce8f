"""GPU parity: attention over packed texts, forward and backward, vs float64.

Tolerances, per element, from arithmetic (h: half a step of the type, 0 for float32 inside):
  O  = sum P V / sum P: every P is rounded, off by h of itself, in the product and in the sum: 2 h sum P |V|; + h |O| (the
                  result);
  dV = sum P dO:  P is rounded, and off as a whole by its row's sum of rounded ones: 2 h sum P |dO|; + h |dV|;
  dS = P (dP - D): P off as a whole by h, D uses the rounded O, off by h sum |dO O|, and dS itself is rounded:
                  e = h (P sum |dO O| + 2 |dS|), so dQ: sum e |K| + h |dQ|, dK: sum e |Q| + h |dK| (scaled);
  float32 sums everywhere: 256 units of 2^-24 (sums of at most that many terms, the exponential's argument with it)
                  of the sum of the terms' sizes."""
import itertools
import math

import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
H = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
bf16, f32 = torch.bfloat16, torch.float32

CASES = [
    # (query lengths, key lengths or None, rows behind, Hq, Hkv, d, window, sinks, dtype)
    ((1,), None, 0, 1, 1, 64, 0, 0, bf16),
    ((0, 1, 2, 0, 3, 0), None, 0, 2, 2, 64, 0, 0, bf16),        # empty texts, also the first and the last
    ((130, 5, 257, 128), None, 0, 4, 2, 128, 0, 0, bf16),       # ends inside, at and past a block
    ((130, 5, 257, 128), None, 7, 4, 1, 64, 0, 0, bf16),        # rows behind the last text
    ((0, 0), None, 40, 2, 1, 64, 0, 0, bf16),                   # nothing but rows behind
    ((200, 61), None, 130, 2, 1, 128, 40, 4, bf16),             # window and sinks
    ((700, 20), None, 0, 2, 1, 128, 256, 70, bf16),             # sinks over a key tile
    ((400, 3), None, 0, 2, 2, 96, 33, 200, bf16),               # more sinks than a key block
    ((190, 140), None, 0, 3, 1, 80, 0, 0, bf16),                # width padded
    ((150, 33), None, 3, 2, 1, 20, 31, 2, bf16),                # rows off 16 bytes
    ((300, 40), None, 0, 4, 2, 32, 1, 1, bf16),                 # the own key and one sink
    ((140, 9), None, 1, 1, 1, 7, 0, 0, f32),
    ((300, 77), None, 0, 4, 2, 64, 0, 0, f32),
    ((270, 1, 64), None, 0, 2, 1, 128, 90, 40, f32),
    ((129, 128), None, 0, 3, 3, 36, 0, 0, f32),
    # queries at the end of longer keys
    ((1, 5, 64, 0), (300, 5, 64, 9), 0, 4, 2, 128, 0, 0, bf16),
    ((33, 130), (700, 131), 4, 8, 2, 64, 0, 0, bf16),
    ((20, 128, 1), (1500, 200, 1), 0, 2, 1, 128, 100, 10, bf16),
    ((40, 3), (513, 90), 0, 4, 4, 64, 0, 0, f32),
    ((2, 50), (400, 60), 0, 2, 1, 72, 64, 3, f32),
    # more queries than keys: the first ones see none
    ((9, 150, 4), (4, 20, 0), 2, 2, 1, 64, 0, 0, bf16),
    ((300, 1), (10, 1), 0, 2, 2, 32, 0, 0, f32),
    # enough blocks that no chunks are made, of each width and type
    (tuple(range(1, 200, 7)), None, 5, 16, 4, 128, 0, 0, bf16),
    (tuple(range(1, 200, 7)), None, 5, 16, 4, 64, 50, 3, bf16),
    (tuple(range(150, 1, -9)), None, 0, 32, 8, 80, 0, 0, bf16),
    (tuple(range(150, 1, -9)), None, 0, 32, 16, 40, 0, 0, bf16),
    (tuple(range(150, 1, -9)), None, 0, 32, 8, 112, 70, 0, bf16),
    (tuple(range(1, 130, 5)), None, 3, 16, 8, 64, 0, 0, f32),
    (tuple(range(1, 130, 5)), None, 3, 16, 8, 128, 40, 2, f32),
    (tuple([1] * 300), None, 0, 4, 2, 64, 0, 0, bf16),          # many texts of one token: the search over offsets in steps
    (tuple([2, 0, 1] * 1500), None, 0, 2, 1, 32, 0, 0, bf16),
]


def _offsets(lengths):
    return list(itertools.accumulate(lengths, initial=0))


def _make(case, seed=0):
    nq, nk, behind, Hq, Hkv, d = case[:6]
    N, M = sum(nq) + behind, sum(nk or nq) + behind
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(h, n, d, generator=g, dtype=torch.float64).to(case[-1]) for h, n in ((Hq, N), (Hkv, M), (Hkv, M), (Hq, N))]


def _within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    ratio = ((got - want).abs() / tol.clamp(min=1e-300)).nan_to_num(0.0)
    assert got.numel() == 0 or bool((ratio <= 1).all()), f"{what}: {float(ratio.max()):.3f} of the tolerance"


def _expected(case, q, k, v, do):
    """(value, tolerance) of O, dQ, dK, dV."""
    nq, nk, behind, Hq, Hkv, d, window, sinks, dtype = case
    G, h, s = Hq // Hkv, H[dtype], d ** -0.5
    q, k, v, do = (t.double() for t in (q, k, v, do))
    want = {"O": torch.zeros_like(q), "dQ": torch.zeros_like(q), "dK": torch.zeros_like(k), "dV": torch.zeros_like(k)}
    tol = {n: torch.zeros_like(t) for n, t in want.items()}
    of = h + 256 * U
    shared = lambda t: t.unflatten(0, (Hkv, G)).sum(1)  # noqa: E731
    for a, b, c, e in zip(*(x for o in (_offsets(nq), _offsets(nk or nq)) for x in (o[:-1], o[1:]))):
        if a == b or c == e:
            continue
        x, y = slice(a, b), slice(c, e)
        qt, dt, kr, vr = q[:, x], do[:, x], k[:, y].repeat_interleave(G, 0), v[:, y].repeat_interleave(G, 0)
        p = od.text_probabilities(qt, k[:, y], window, sinks)
        o = p @ vr
        ds = p * (dt @ vr.transpose(-1, -2) - (dt * o).sum(-1, keepdim=True))
        size = p * (dt.abs() @ vr.abs().transpose(-1, -2) + (dt * o).abs().sum(-1, keepdim=True))
        err = h * (p * (dt * o).abs().sum(-1, keepdim=True) + 2 * ds.abs()) + 256 * U * size
        want["O"][:, x], tol["O"][:, x] = o, (of + h) * (p @ vr.abs())
        want["dQ"][:, x], tol["dQ"][:, x] = s * ds @ kr, s * err @ kr.abs()
        want["dK"][:, y], tol["dK"][:, y] = (s * shared(ds.transpose(-1, -2) @ qt), s * shared(err.transpose(-1, -2) @ qt.abs()))
        want["dV"][:, y], tol["dV"][:, y] = (shared(p.transpose(-1, -2) @ dt), (of + h) * shared(p.transpose(-1, -2) @ dt.abs()))
    return {n: (want[n], tol[n] + max(h, U) * want[n].abs()) for n in want}


def _dev(offsets):
    return torch.tensor(offsets, dtype=torch.int32).cuda()


def _name(case):
    nq, nk = case[:2]
    texts = "x".join(map(str, nq)) if len(nq) < 9 else f"{len(nq)}texts{sum(nq)}"
    return texts + ("of" + "x".join(map(str, nk)) if nk else "") + "-" + "-".join(str(x).replace("torch.", "") for x in case[2:])


@pytest.mark.parametrize("case", CASES, ids=_name)
def test_packed_attention_fwd_bwd(case):
    from edifice_amd import fused_scan as fs
    nq, nk, behind, Hq, Hkv, d, window, sinks, dtype = case
    announce("packed_attention", case=case if len(nq) < 40 else case[2:])
    q, k, v, do = _make(case)
    qo, ko = _dev(_offsets(nq)), _dev(_offsets(nk)) if nk else None
    tq, tk, tv = (t.cuda().requires_grad_() for t in (q, k, v))
    out = fs.packed_attention(tq, tk, tv, qo, ko, window=window, sinks=sinks)
    grads = torch.autograd.grad(out, (tq, tk, tv), do.cuda())
    again = torch.autograd.grad(fs.packed_attention(tq, tk, tv, qo, ko, window=window, sinks=sinks), (tq, tk, tv), do.cuda())
    exp = _expected(case, q, k, v, do)
    for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
        _within(got, *exp[name], name)
    for a, b in zip(grads, again):  # sums in a fixed order
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(fs.packed_attention(tq, tk, tv, qo, ko, window=window, sinks=sinks), out)


@pytest.mark.parametrize("case", [
    # few queries' key tiles in chunks, of each width and type
    ((400, 303), None, 5, 2, 1, 32, 0, 0, bf16),
    ((520, 1, 90), None, 0, 3, 3, 96, 70, 100, bf16),
    ((30, 2), (900, 300), 0, 4, 2, 80, 0, 0, bf16),
    ((600, 33), None, 3, 2, 1, 20, 0, 2, bf16),
    ((40, 300), (600, 300), 0, 4, 1, 112, 0, 0, bf16),
    ((250, 9), None, 1, 1, 1, 7, 0, 0, f32),
    ((210, 60), None, 0, 2, 2, 100, 0, 0, f32),
    ((5, 200), (500, 210), 2, 8, 2, 30, 150, 1, f32),
    # and as many keys as are not cut
    ((300, 212), None, 0, 2, 1, 64, 0, 0, bf16),
    ((300, 213), None, 0, 2, 1, 128, 0, 0, bf16),
    ((150, 42), None, 0, 2, 2, 64, 0, 0, f32),
    ((150, 43), None, 0, 2, 2, 128, 0, 0, f32),
], ids=_name)
def test_chunks_of_each_width(case):
    test_packed_attention_fwd_bwd(case)


def test_texts_do_not_reach_one_another():
    """Values of one text that are not finite leave the others as they were, forward and backward."""
    from edifice_amd import fused_scan as fs
    announce("packed, texts apart")
    case = ((150, 70, 200), None, 30, 4, 2, 128, 0, 0, bf16)
    for case in (case, case[:5] + (64,) + case[6:8] + (f32,), case[:5] + (20,) + case[6:]):
        q, k, v, do = (t.cuda() for t in _make(case))
        off = _dev(_offsets(case[0]))

        def call():
            leaves = [t.clone().requires_grad_() for t in (q, k, v)]
            o = fs.packed_attention(*leaves, off)
            return [o, *torch.autograd.grad(o, leaves, do)]

        want = call()
        for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (do, math.inf)):
            t[:, 150:220] = bad
            t[:, 420:] = bad  # behind the last text
        for got, ref in zip(call(), want):
            assert torch.equal(got[:, :150], ref[:, :150]) and torch.equal(got[:, 220:420], ref[:, 220:420])
            assert not got[:, 420:].any()


def test_offsets_out_of_order_stay_in_bounds():
    """Offsets that do not ascend, or lead past the rows, are clamped: the call ends, and texts that are right stay so."""
    from edifice_amd import fused_scan as fs
    announce("packed, offsets out of order")
    q, k, v, do = (t.cuda() for t in _make(((300,), None, 0, 2, 1, 64, 0, 0, bf16)))
    right = fs.packed_attention(q, k, v, _dev([0, 150, 300]))
    for offsets in ([0, 150, 900], [0, 150, 2 ** 31 - 1], [5, 150, 300]):
        assert torch.equal(fs.packed_attention(q, k, v, _dev(offsets)), right)
    for offsets in ([0, 200, 100], [0, -5, -7], [0, 2 ** 31 - 1, -2 ** 31], [0, 299, 5, 290, 8]):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = fs.packed_attention(*leaves, _dev(offsets))
        torch.autograd.grad(o, leaves, do)
        torch.cuda.synchronize()


def test_gradients_against_differences():
    """Central differences of the float32 forward along random directions."""
    from edifice_amd import fused_scan as fs
    announce("packed, differences")
    case = ((50, 7, 140), (90, 7, 150), 0, 4, 2, 48, 30, 4, f32)
    q, k, v, do = (t.cuda() for t in _make(case, 3))
    qo, ko = _dev(_offsets(case[0])), _dev(_offsets(case[1]))
    loss = lambda *x: (fs.packed_attention(*x, qo, ko, window=30, sinks=4).double() * do.double()).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    g = torch.Generator().manual_seed(4)
    for i, grad in enumerate(grads):
        u = torch.randn(grad.shape, generator=g).cuda()
        step = 2.0 ** -6
        with torch.no_grad():
            ends = [loss(*(t + sign * step * u if j == i else t for j, t in enumerate((q, k, v)))) for sign in (1, -1)]
        slope, want = (ends[0] - ends[1]) / (2 * step), (grad.double() * u.double()).sum()
        # the third derivative's share step^2 / 6, of order one relative to the gradients' size, and float32's rounding of
        # the two sums of products of size one, U sqrt(terms) / step
        size = (grad.double() * u.double()).norm()
        assert abs(float(slope - want)) <= float(size) * step ** 2 * 4 + 16 * U * do.numel() ** 0.5 / step


def test_captured_and_replayed_with_other_offsets():
    """Forward and backward in one graph; the offsets change between replays, eager work lies between them."""
    from edifice_amd import fused_scan as fs
    announce("packed, captured")
    g = torch.Generator().manual_seed(5)
    for Hq, Hkv, d, dtype in ((4, 2, 128, bf16), (4, 4, 64, f32)):
        q, k, v, do = (torch.randn(h, 400, d, generator=g).to(dtype).cuda() for h in (Hq, Hkv, Hkv, Hq))
        off = _dev([0, 100, 250, 400])

        def step():
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            o = fs.packed_attention(*leaves, off)
            return [o.detach(), *torch.autograd.grad(o, leaves, do)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for offsets in ([0, 400, 400, 400], [0, 1, 2, 390], [0, 0, 399, 400], [0, 133, 140, 300]):
            off.copy_(_dev(offsets))
            q.copy_(torch.randn(q.shape, generator=g))
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), offsets


def test_layouts_and_streams():
    """[1, H, N, d] as the head split gives it, strided inputs, and a stream other than the tensors' own."""
    from edifice_amd import fused_scan as fs
    announce("packed, layouts")
    case = ((120, 30), None, 10, 4, 2, 64, 0, 0, bf16)
    q, k, v, do = (t.cuda() for t in _make(case))
    off = _dev([0, 120, 150])
    want = fs.packed_attention(q, k, v, off)
    assert torch.equal(fs.packed_attention(q[None], k[None], v[None], off)[0], want)
    wide = torch.empty(160, 4, 64, device="cuda", dtype=bf16).copy_(q.transpose(0, 1))
    assert torch.equal(fs.packed_attention(wide.transpose(0, 1), k, v, off), want)
    off16 = torch.empty(4 * 160 * 64 + 1, device="cuda", dtype=bf16)[1:].view(4, 160, 64).copy_(q)  # 2 bytes off 16
    _within(fs.packed_attention(off16, k, v, off), want.cpu().double(), 2.0 ** -6 * want.abs().cpu().double() + 2.0 ** -6, "O")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = fs.packed_attention(*leaves, off)
        o.backward(do)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want)


def test_empty_and_broadcast():
    from edifice_amd import fused_scan as fs
    announce("packed, empty")
    off = _dev([0, 0])
    q, k = torch.zeros(2, 0, 8).cuda().requires_grad_(), torch.zeros(1, 0, 8).cuda()
    assert fs.packed_attention(q, k, k, off).shape == (2, 0, 8)
    q = torch.randn(2, 3, 8).cuda().requires_grad_()
    o = fs.packed_attention(q, k, k, _dev([0, 3]), off)  # queries without keys
    o.sum().backward()
    assert not o.any() and not q.grad.any()
    o = fs.packed_attention(q, q[:1], q[:1], _dev([0]))  # no text
    assert not o.any()
    # one key and value for both heads, and a gradient that is one number broadcast
    k = torch.randn(1, 3, 8).cuda().requires_grad_()
    o = fs.packed_attention(q, k.expand(2, 3, 8), k.expand(2, 3, 8), _dev([0, 2, 3]))
    o.sum().backward()
    want = fs.packed_attention(q.detach(), k.detach(), k.detach(), _dev([0, 2, 3]))
    assert torch.allclose(o, want, atol=1e-6) and k.grad.shape == k.shape


def test_a_long_text():
    """The last queries of a text whose heads pass 2^31 bytes together, against the keys that they see."""
    from edifice_amd import fused_scan as fs
    announce("packed, long")
    N, d, window = 70000, 128, 300
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(140, N, d, generator=g, device="cuda", dtype=bf16)  # 2.5 GB
    k, v = (torch.randn(70, N, d, generator=g, device="cuda", dtype=bf16) for _ in range(2))
    out = fs.packed_attention(q, k, v, _dev([0, 123, N]), window=window, sinks=2)
    for h, i in itertools.product((0, 77, 139), (0, 122, 123, 5000, N - 1)):
        first = 0 if i < 123 else 123
        js = [j for j in range(first, i + 1) if i - j < window or j - first < 2]
        kj, vj = k[h // 2, js].double(), v[h // 2, js].double()
        p = torch.softmax(kj @ q[h, i].double() / math.sqrt(d), 0)
        _within(out[h, i], (p @ vj).cpu(), ((2.0 ** -7 + 256 * U) * (p @ vj.abs()) + 2.0 ** -8 * (p @ vj).abs()).cpu(), f"{h} {i}")


@pytest.mark.parametrize("M, d", [((1 << 22) - 1, 128), (4300001, 64)], ids=["rows in pieces", "rows by element"])
def test_keys_past_two_to_the_31_bytes(M, d):
    """A text of a few queries on so many keys that its heads pass 2^31 bytes, and one behind it, forward and backward."""
    from edifice_amd import fused_scan as fs
    announce("packed, long keys", M=M, d=d)
    first, n = M - 300, 20
    g = torch.Generator(device="cuda").manual_seed(8)
    q, do = (torch.randn(4, n + 5, d, generator=g, device="cuda", dtype=bf16) for _ in range(2))
    k, v = (torch.randn(4, M, d, generator=g, device="cuda", dtype=bf16) for _ in range(2))  # 4.3 and 2.2 GB
    # query 3 of the first text finds a key near its end, so far above the rest that P is 1 there
    at = first - n - 100
    q[:, 3] = torch.randn(d, generator=g, device="cuda").sign()
    k[:, at] = 8 * q[:, 3]
    qo, ko = _dev([0, n, n + 5]), _dev([0, first, M])
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = fs.packed_attention(*leaves, qo, ko)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    # scores of query 3: 8 sqrt(d) >= 64 against |q . k| / sqrt(d) <= 6.5 or so of M random ones: exp(-57) M is nothing
    assert torch.equal(out[:, 3], v[:, at])
    # dV there: dO of query 3, and P of the others.  Their scores at that key are sums of d float32 terms of 8 |q| / sqrt(d), 72
    # together: off by d U 72 < 2^-10.8 here and in the kernel, twice over with the row sums: 2^-8
    with torch.no_grad():
        p = torch.zeros(4, n, dtype=torch.float64, device="cuda")
        for h in range(4):
            s = torch.cat([c.float() @ q[h, :n].float().T for c in k[h, :first].split(1 << 20)]).double() / math.sqrt(d)
            s.masked_fill_(torch.arange(first, device="cuda")[:, None] > torch.arange(first - n, first, device="cuda"), -math.inf)
            p[h] = torch.softmax(s, 0)[at]
        want = (p[..., None] * do[:, :n].double()).sum(1)
        size = (p[..., None] * do[:, :n].double().abs()).sum(1)
    _within(dv[:, at], want.cpu(), ((2.0 ** -7 + 256 * U + 2.0 ** -8) * size + 2.0 ** -8 * want.abs()).cpu(), "dV")
    case = ((5,), (300,), 0, 4, 4, d, 0, 0, bf16)
    exp = _expected(case, *(t.detach().cpu() for t in (q[:, n:], k[:, first:], v[:, first:], do[:, n:])))
    for name, got in (("O", out[:, n:]), ("dQ", dq[:, n:]), ("dK", dk[:, first:]), ("dV", dv[:, first:])):
        _within(got, *exp[name], name)
