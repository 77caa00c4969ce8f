"""GPU parity: attention with a window and sinks, forward and backward, vs float64.

Tolerances, per element, from arithmetic (h: half a step of the type, 0 for float32 inside):
  O  = sum P V / sum P: every P is rounded, off by h of itself, in the product and, where the kernel sums what it
                  multiplies, in the sum: sum P (d_j - mean d) V with |d_j| <= h, so 2 h sum P |V|; + h |O| (the result);
  dV = sum P dO:  h sum P |dO| + h |dV|;
  dS = P (dP - D): D uses the rounded O, off by h sum |dO O|; dS itself is rounded:
                  e = P h sum |dO O| + h |dS|, so dQ: sum e |K| + h |dQ|, dK: sum e |Q| + h |dK| (scaled);
  float32 sums everywhere: 256 units of 2^-24 (sums of at most that many terms, the exponential's argument with it)
                  of the sum of the terms' sizes."""
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
    # (B, Hq, Hkv, T, d, window, sinks, dtype)
    (1, 1, 1, 1, 64, 1, 0, bf16),        # one token
    (2, 4, 2, 2, 64, 2, 0, bf16),
    (1, 4, 1, 130, 128, 40, 4, bf16),    # window inside a tile, a block of two queries at the end
    (2, 2, 2, 300, 128, 128, 0, bf16),
    (1, 8, 2, 513, 64, 200, 3, bf16),
    (1, 2, 1, 700, 128, 256, 70, bf16),  # sinks over a key tile
    (1, 2, 2, 200, 32, 1000, 0, bf16),   # window past the sequence: causal
    (1, 2, 1, 260, 32, 1, 1, bf16),      # the own key and one sink
    (1, 2, 2, 400, 96, 33, 200, bf16),   # more sinks than a key block
    (1, 3, 1, 190, 80, 64, 5, bf16),     # width padded
    (1, 2, 1, 150, 20, 31, 2, bf16),     # rows off 16 bytes
    (1, 1, 1, 140, 7, 31, 2, f32),
    (2, 4, 2, 300, 64, 100, 1, f32),
    (1, 2, 1, 270, 128, 90, 40, f32),
    (1, 3, 3, 129, 36, 129, 0, f32),
    (1, 6, 2, 1100, 64, 96, 2, f32),     # several workgroups share a sink block
    # grids of 160 blocks of 128 queries and more: the wide kernels of each width and type
    (10, 8, 2, 135, 32, 20, 3, bf16),
    (10, 8, 4, 200, 64, 70, 4, bf16),
    (5, 16, 8, 300, 64, 1000, 0, bf16),
    (10, 8, 2, 150, 80, 64, 1, bf16),
    (10, 8, 8, 140, 96, 33, 20, bf16),
    (10, 8, 2, 150, 112, 60, 2, bf16),
    (10, 8, 2, 140, 52, 60, 2, bf16),
    (10, 8, 2, 200, 128, 100, 5, bf16),
    (3, 16, 4, 520, 128, 130, 70, bf16),
    (10, 8, 2, 135, 32, 200, 0, f32),
    (10, 8, 4, 150, 64, 40, 4, f32),
    (10, 8, 2, 135, 72, 30, 2, f32),
    (10, 8, 4, 140, 128, 64, 1, f32),
]


def _make(case, seed=0):
    B, Hq, Hkv, T, d, window, sinks, dtype = case
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, h, T, d, generator=g, dtype=torch.float64).to(dtype) for h in (Hq, Hkv, Hkv, Hq)]


def _within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    ratio = ((got - want).abs() / tol.clamp(min=1e-300)).nan_to_num(0.0)
    assert bool((ratio <= 1).all()), f"{what}: {float(ratio.max()):.3f} of the tolerance"


def _expected(case, q, k, v, do):
    """(value, tolerance) of O, dQ, dK, dV."""
    B, Hq, Hkv, T, d, window, sinks, dtype = case
    G, h, s = Hq // Hkv, H[dtype], d ** -0.5
    q, k, v, do = (t.double() for t in (q, k, v, do))
    kr, vr = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    p = od.window_probabilities(q, k, window, sinks)
    o = p @ vr
    dp = do @ vr.transpose(-1, -2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    shared = lambda t: t.view(B, Hkv, G, T, d).sum(2)  # noqa: E731
    pt, dst = p.transpose(-1, -2), ds.transpose(-1, -2)
    # sizes of dS's terms: the two float32 dot products behind it
    size = p * (do.abs() @ vr.abs().transpose(-1, -2) + (do * o).abs().sum(-1, keepdim=True))
    e = h * (p * (do * o).abs().sum(-1, keepdim=True) + ds.abs()) + 256 * U * size
    et = e.transpose(-1, -2)
    of = (h + 256 * U)
    want = {"O": o, "dQ": s * ds @ kr, "dK": s * shared(dst @ q), "dV": shared(pt @ do)}
    tol = {"O": (of + h) * (p @ vr.abs()), "dQ": s * e @ kr.abs(), "dK": s * shared(et @ q.abs()),
           "dV": of * shared(pt @ do.abs())}
    return {n: (want[n], tol[n] + max(h, U) * want[n].abs()) for n in want}


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_window_attention_fwd_bwd(case):
    from edifice_amd import fused_scan as fs
    B, Hq, Hkv, T, d, window, sinks, dtype = case
    announce("window_attention", case=case)
    q, k, v, do = _make(case)
    tq, tk, tv = (t.cuda().requires_grad_() for t in (q, k, v))
    out = fs.window_attention(tq, tk, tv, window, sinks)
    grads = torch.autograd.grad(out, (tq, tk, tv), do.cuda())
    again = torch.autograd.grad(fs.window_attention(tq, tk, tv, window, sinks), (tq, tk, tv), do.cuda())
    exp = _expected(case, q, k, v, do)
    for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
        _within(got, *exp[name], name)
    for a, b in zip(grads, again):  # sums in a fixed order
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(fs.window_attention(tq, tk, tv, window, sinks), out)


def test_far_queries_against_a_band():
    """A long sequence: its last queries against the keys that they see (offsets past the first tiles, many blocks)."""
    from edifice_amd import fused_scan as fs
    announce("window_long")
    B, Hq, Hkv, T, d, window, sinks = 1, 2, 1, 9000, 64, 500, 4
    q, k, v, _ = _make((B, Hq, Hkv, T, d, window, sinks, bf16))
    out = fs.window_attention(q.cuda(), k.cuda(), v.cuda(), window, sinks).cpu().double()
    for i in (0, 3, 4, 499, 500, 505, 4321, 8191, 8999):
        js = [j for j in range(i + 1) if i - j < window or j < sinks]
        kj, vj = k[0, 0, js].double(), v[0, 0, js].double()
        for h in range(Hq):
            p = torch.softmax(kj @ q[0, h, i].double() / math.sqrt(d), 0)
            _within(out[0, h, i], p @ vj, (2.0 ** -7 + 256 * U) * (p @ vj.abs()) + 2.0 ** -8 * (p @ vj).abs(), f"row {i}")


def _banded(q, k, v, do, window, sinks, h):
    """_expected for one query head [T, d] of a long sequence and a short window, from the keys that each query sees."""
    T, d = q.shape
    q, k, v, do = (t.double() for t in (q, k, v, do))
    i = torch.arange(T, device=q.device)[:, None]
    near, sink = i - torch.arange(window, device=q.device), torch.arange(sinks, device=q.device).expand(T, sinks)
    idx = torch.cat([near.clamp(min=0), sink], 1)
    seen = torch.cat([near >= 0, sink <= i - window], 1)
    kj, vj, s = k[idx], v[idx], d ** -0.5
    p = torch.softmax(((kj * q[:, None]).sum(-1) * s).masked_fill(~seen, -math.inf), 1)
    o = (p[..., None] * vj).sum(1)
    dp, dd = (vj * do[:, None]).sum(-1), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dd)
    size = p * ((vj.abs() * do.abs()[:, None]).sum(-1) + (do * o).abs().sum(-1, keepdim=True))
    e = h * (p * (do * o).abs().sum(-1, keepdim=True) + ds.abs()) + 256 * U * size
    # a sink's sums: fewer than 2048 additions, one after another, in a wave, between waves and between workgroups
    n = 2048 * U
    back = lambda w, x: torch.zeros_like(k).index_add_(0, idx.flatten(), (w[..., None] * x[:, None]).flatten(0, 1))  # noqa: E731
    return ((s * back(ds, q), s * back(e + n * ds.abs(), q.abs())), (back(p, do), (h + n) * back(p, do.abs())),
            (s * (ds[..., None] * kj).sum(1), s * (e[..., None] * kj.abs()).sum(1)))


@pytest.mark.parametrize("case", [(1, 8, 1, 6000, 32, bf16, 0, 3), (1, 128, 8, 8192, 32, bf16, 0, 3), (1, 128, 8, 8192, 32, bf16, 1, 3),
                                  (2, 32, 4, 6000, 64, bf16, 0, 3), (2, 32, 4, 6000, 64, bf16, 0, 40), (2, 32, 4, 6001, 64, bf16, 1, 3),
                                  (1, 128, 8, 8192, 88, bf16, 0, 3), (1, 128, 8, 8180, 88, bf16, 1, 3),
                                  (2, 32, 4, 6000, 128, bf16, 0, 3), (2, 32, 4, 6000, 128, bf16, 1, 3),
                                  (2, 16, 2, 6000, 32, f32, 0, 3), (2, 16, 2, 6000, 32, f32, 1, 40), (1, 8, 1, 6001, 64, f32, 0, 40),
                                  (1, 8, 1, 6000, 64, f32, 1, 3), (1, 8, 2, 6000, 84, f32, 0, 3), (1, 8, 2, 6000, 84, f32, 1, 3),
                                  (1, 8, 1, 5999, 128, f32, 0, 140), (1, 8, 1, 3000, 126, f32, 0, 3)], ids=str)
def test_sinks_of_a_long_sequence(case):
    """dK and dV of sinks that thousands of queries see past their windows, in the calls that give these queries a
    kernel of their own and those that do not; tensors whole 16 bytes or one element off them."""
    from edifice_amd import fused_scan as fs
    B, Hq, Hkv, T, d, dtype, off, sinks = case
    announce("window_sinks", case=case)
    window, g = 9, torch.Generator(device="cuda").manual_seed(sinks)

    def make(H_):
        buf = torch.randn(B * H_ * T * d + off, device="cuda", generator=g, dtype=torch.float32).to(dtype)
        return buf[off:].view(B, H_, T, d)
    q, k, v, do = (make(n) for n in (Hq, Hkv, Hkv, Hq))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(fs.window_attention(q, k, v, window, sinks), leaves, do)
    G, half = Hq // Hkv, max(H[dtype], U)
    b, kh = B - 1, Hkv - 1
    heads = [_banded(*(t.detach()[b, h] for t, h in ((q, h), (k, kh), (v, kh), (do, h))), window, sinks, H[dtype])
             for h in range(kh * G, (kh + 1) * G)]
    for x, got, name in ((0, dk, "dK"), (1, dv, "dV")):
        want, tol = (sum(h[x][y] for h in heads) for y in (0, 1))
        _within(got[b, kh], want.cpu(), (tol + half * want.abs()).cpu(), name)
    want, tol = heads[-1][2]
    _within(dq[b, -1], want.cpu(), (tol + half * want.abs()).cpu(), "dQ")


@pytest.mark.parametrize("T, d, dtype", [((1 << 22) - 1, 128, bf16), ((1 << 22) - 1, 128, f32), ((1 << 22) + 70, 128, f32),
                                         ((1 << 22) + 70, 64, bf16)], ids=str)
def test_the_end_of_a_very_long_sequence(T, d, dtype):
    """Offsets up to and past 2^31 bytes of one head: without sinks the last tokens are a sequence of their own."""
    from edifice_amd import fused_scan as fs
    announce("window_very_long", T=T, d=d, dtype=dtype)
    window, last = 50, 400
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(1, 1, T, d, device="cuda", generator=g, dtype=dtype) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = fs.window_attention(q, k, v, window)
    grads = torch.autograd.grad(out, leaves, do)
    exp = _expected((1, 1, 1, last, d, window, 0, dtype), *(t.detach()[:, :, -last:].cpu() for t in (q, k, v, do)))
    for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
        # from here on every query's keys, and every key's queries', lie in the piece
        _within(got[:, :, -(last - window):], *(t[:, :, window:] for t in exp[name]), name)


def test_causal_window_matches_flash_attention():
    """window >= T, one key head per query head: the causal flash kernel's result to their roundings."""
    from edifice_amd import fused_scan as fs
    announce("window_flash")
    case = (1, 2, 2, 333, 128, 333, 0, bf16)
    q, k, v, do = _make(case)
    got = fs.window_attention(q.cuda(), k.cuda(), v.cuda(), 333)
    want = fs.flash_attention(q.cuda(), k.cuda(), v.cuda(), causal=True)
    tol = _expected(case, q, k, v, do)["O"][1]
    _within(got, want.cpu().double(), 2 * tol, "flash")


def test_a_window_without_end():
    """A window and sinks past any int are those of the whole length, not their low bits."""
    from edifice_amd import fused_scan as fs
    announce("window_without_end")
    q, k, v, _ = _make((1, 4, 2, 77, 64, 77, 0, bf16))
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    want = fs.window_attention(q, k, v, 77)
    assert torch.equal(fs.window_attention(q, k, v, 2**63 - 1), want)
    assert torch.equal(fs.window_attention(q, k, v, 2**32 + 3), want)
    assert torch.equal(fs.window_attention(q, k, v, 77, 2**32 + 3), want)


def test_many_heads():
    """More heads than a grid's second axis holds, and sinks whose gradients are divided."""
    from edifice_amd import fused_scan as fs
    announce("window_many_heads")
    B, H, T, d = 1100, 64, 40, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(B, H, T, d, device="cuda", generator=g) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = fs.window_attention(q, k, v, 7, 2)
    grads = torch.autograd.grad(out, leaves, do)
    for b, h in ((0, 0), (1023, 63), (1099, 63)):
        one = [t.detach()[b:b + 1, h:h + 1].cpu() for t in (q, k, v, do)]
        exp = _expected((1, 1, 1, T, d, 7, 2, f32), *one)
        for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
            _within(got[b:b + 1, h:h + 1], *exp[name], f"{name} of head {b}, {h}")


def test_strided_and_broadcast_inputs():
    """Head-interleaved views and a key head expanded to several are copied, and their gradients are summed back."""
    from edifice_amd import fused_scan as fs
    announce("window_strides")
    case = (1, 4, 2, 70, 32, 20, 1, f32)
    q, k, v, do = _make(case)
    qi = q.transpose(1, 2).contiguous().cuda().requires_grad_()
    k1 = k[:, :1].cuda().requires_grad_()
    out = fs.window_attention(qi.transpose(1, 2), k1.expand(1, 2, 70, 32), v.cuda(), 20, 1)
    dq, dk = torch.autograd.grad(out, (qi, k1), do.cuda())
    exp = _expected(case, q, k[:, :1].expand(1, 2, 70, 32), v, do)
    _within(out, *exp["O"], "O")
    _within(dq.transpose(1, 2), *exp["dQ"], "dQ")
    _within(dk, exp["dK"][0].sum(1, keepdim=True), exp["dK"][1].sum(1, keepdim=True), "dK")


@pytest.mark.parametrize("case", [(1, 4, 2, 300, 128, 90, 3, bf16), (1, 4, 1, 200, 64, 70, 2, bf16),
                                  (2, 2, 1, 150, 96, 40, 0, bf16), (1, 2, 1, 170, 64, 50, 1, f32),
                                  (1, 2, 2, 140, 128, 64, 2, f32), (10, 8, 2, 150, 128, 60, 2, bf16)], ids=str)
def test_tensors_one_element_off(case):
    """Contiguous tensors whose rows are off 16 bytes, in and for the gradient of the result."""
    from edifice_amd import fused_scan as fs
    announce("window_off", case=case)

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)
    q, k, v, do = _make(case)
    leaves = [off(t).requires_grad_() for t in (q, k, v)]
    out = fs.window_attention(*leaves, *case[5:7])
    grads = torch.autograd.grad(out, leaves, off(do))
    exp = _expected(case, q, k, v, do)
    for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
        _within(got, *exp[name], name)


def test_extreme_scores():
    """Scores far apart (one key takes all) and large equal ones: finite, and the softmax of the definition."""
    from edifice_amd import fused_scan as fs
    announce("window_extreme")
    case = (1, 1, 1, 96, 64, 50, 1, f32)
    q, k, v, do = _make(case)
    k = k * 100
    k[0, 0, 10] = q[0, 0, 10] * 1000
    tq, tk, tv = (t.cuda().requires_grad_() for t in (q, k, v))
    out = fs.window_attention(tq, tk, tv, 50, 1)
    grads = torch.autograd.grad(out, (tq, tk, tv), do.cuda())
    p = od.window_probabilities(q.double(), k.double(), 50, 1)
    # a score of size s has a float32 error of 64 units of s, which moves P by that much relative to itself
    s = (q.double().abs() @ k.double().abs().transpose(-1, -2) / 8).amax(-1, keepdim=True)
    tol = (256 + 128 * s) * U * (p @ v.double().abs()) + 128 * s * U * v.double().abs().amax()
    _within(out, p @ v.double(), tol, "O")
    assert all(torch.isfinite(g).all() for g in grads)


def test_side_stream():
    """The call runs on the current stream."""
    from edifice_amd import fused_scan as fs
    announce("window_stream")
    q, k, v, _ = (t.cuda() for t in _make((1, 2, 1, 200, 64, 50, 2, bf16)))
    want = fs.window_attention(q, k, v, 50, 2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = fs.window_attention(q, k, v, 50, 2)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("case", [(1, 4, 2, 300, 64, 100, 2, bf16), (1, 8, 1, 6001, 64, 9, 40, f32)], ids=str)
def test_captured_forward_and_backward(case):
    """Forward and backward through the C entry points in one graph, replayed on new contents."""
    from edifice_amd import fused_scan as fs
    announce("window_graph", case=case)
    B, Hq, Hkv, T, d, window, sinks, dtype = case
    st = [t.cuda() for t in _make(case)]

    def step():
        q, k, v = (t.detach().requires_grad_() for t in st[:3])
        out = fs.window_attention(q, k, v, window, sinks)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), st[3])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(1, 4):
        for t, n in zip(st, _make(case, seed)):
            t.copy_(n)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """sum(do . O) along a direction, central differences of the float64 form against the kernel's gradients."""
    from edifice_amd import fused_scan as fs
    announce("window_differences")
    case = (1, 4, 2, 90, 32, 25, 2, f32)
    q, k, v, do = _make(case)
    tq, tk, tv = (t.cuda().requires_grad_() for t in (q, k, v))
    grads = torch.autograd.grad(fs.window_attention(tq, tk, tv, 25, 2), (tq, tk, tv), do.cuda())
    gen = torch.Generator().manual_seed(5)
    dirs = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (q, k, v)]
    f = lambda e: (od.window_attention(*(t.double() + e * u for t, u in zip((q, k, v), dirs)), 25, 2) * do.double()).sum()  # noqa: E731
    want = float((f(1e-5) - f(-1e-5)) / 2e-5)
    got = sum(float((g.cpu().double() * u).sum()) for g, u in zip(grads, dirs))
    size = sum(float((g.cpu().double() * u).abs().sum()) for g, u in zip(grads, dirs))
    assert abs(got - want) <= 1e-5 * size
