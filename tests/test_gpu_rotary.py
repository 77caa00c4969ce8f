"""GPU parity: the head split with norms and rotary positions, forward and backward, vs float64.

Tolerances, per element, from arithmetic: one rounding of the result, h = eps / 2 of its type relative to it (bf16
2^-8, f32 2^-24), and the float32 inside: the angle's fraction of a turn (2^-25 turns is 1.9e-7 rad, 3 units of
2^-24), the sine (2 units), a sum of squares of at most 256 terms in 16-term lanes (under 24 units), the square
root and four products: under 64 units of 2^-24 of the row's largest element.  The weight gradients add rows * heads
products in float32: sqrt-free, at most (rows + 64) units of the sum of their sizes."""
import math

import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
H = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}

CASES = [
    # (B, T, Hq, Hkv, d, rot, interleaved, norm, amplitude, dtype)
    (2, 33, 8, 2, 128, 128, False, True, 1.0, torch.bfloat16),
    (1, 1, 4, 4, 64, 64, True, True, 1.3, torch.bfloat16),     # one token
    (3, 7, 3, 1, 96, 48, True, False, 1.0, torch.bfloat16),    # part of the head, no norms
    (2, 5, 5, 1, 80, 40, False, True, 1.0, torch.bfloat16),    # half of 20: 8-byte chunks
    (2, 9, 2, 2, 20, 20, False, True, 1.0, torch.bfloat16),    # half of 10: single elements
    (1, 6, 2, 1, 7, 6, True, True, 1.0, torch.bfloat16),       # odd width: the last element has no partner
    (1, 6, 2, 1, 7, 2, False, True, 1.0, torch.float32),
    (2, 70, 4, 2, 256, 256, False, True, 1.0, torch.float32),
    (2, 11, 6, 3, 255, 254, False, True, 0.7, torch.bfloat16),  # widest odd: two units a lane
    (1, 40, 12, 4, 96, 48, True, True, 1.2, torch.float32),
    (2, 13, 4, 1, 64, 0, False, True, 1.0, torch.float32),     # norms alone
    (1, 3, 40, 20, 128, 64, False, True, 1.0, torch.bfloat16),  # more heads than rows of a pass
]


def _make(case, seed=0, positions="far"):
    B, T, Hq, Hkv, d, rot, inter, norm, amp, dtype = case
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
    x = n(B, T, (Hq + 2 * Hkv) * d)
    w = [(1 + 0.3 * torch.randn(d, generator=g, dtype=torch.float64)).to(dtype) if norm else None for _ in range(2)]
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot) if rot else None
    pos = torch.randint(0, 1 << 20, (B, T), generator=g, dtype=torch.int32) if positions == "far" else None
    grads = [n(B, h, T, d) for h in (Hq, Hkv, Hkv)]
    return x, w, freq, pos, grads


def _double(t, grad=True):
    return None if t is None else t.double().requires_grad_(grad)


def _run(case, x, w, freq, pos, grads=None):
    from edifice_amd import fused_scan as fs
    B, T, Hq, Hkv, d, rot, inter, norm, amp, dtype = case
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    xd, wq, wk = dev(x), dev(w[0]), dev(w[1])
    leaves = [t for t in (xd, wq, wk) if t is not None]
    if grads is not None:
        for t in leaves:
            t.requires_grad_()
    out = fs.split_heads_rotary(xd, Hq, Hkv, dev(freq), dev(pos), wq, wk, interleaved=inter, amplitude=amp)
    if grads is None:
        return out
    return [o.detach() for o in out], torch.autograd.grad(out, leaves, [dev(t) for t in grads])


def _check(got, want, dtype, size, what, units=64):
    err = (got.detach().cpu().double() - want).abs()
    tol = H[dtype] * want.abs() + units * U * size
    assert torch.isfinite(got).all() and bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.3f} of the tolerance"


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_split_heads_rotary_fwd_bwd(case):
    B, T, Hq, Hkv, d, rot, inter, norm, amp, dtype = case
    announce("split_heads_rotary", case=case)
    x, w, freq, pos, grads = _make(case)
    out, dev_grads = _run(case, x, w, freq, pos, grads)
    leaves = [_double(x), _double(w[0]), _double(w[1])]
    ref = od.split_heads_rotary(leaves[0], Hq, Hkv, freq, pos, leaves[1], leaves[2], 1e-6, inter, amp)
    for name, o, r in zip("qk", out, ref):
        _check(o, r.detach(), dtype, max(amp, 1) * 1.5 * r.detach().abs().amax(-1, keepdim=True), name)
    assert torch.equal(out[2].cpu(), ref[2].to(dtype))  # v is only moved
    gr = torch.autograd.grad(ref, [t for t in leaves if t is not None], [t.double() for t in grads])
    # dx of a row: a few terms of the row's size each; its largest times d^(1/2) bounds |gw . xh| / d
    row = gr[0].view(B, T, -1, d).abs().amax(-1, keepdim=True).expand(B, T, -1, d).reshape(gr[0].shape)
    _check(dev_grads[0], gr[0], dtype, 4 * row + 1e-3, "dx")
    if norm:
        for i, name, h, at in ((1, "dwq", Hq, 0), (2, "dwk", Hkv, Hq)):
            u = x.double().view(B, T, -1, d)[:, :, at:at + h].transpose(1, 2)
            xh = u / torch.sqrt(u.square().mean(-1, keepdim=True) + 1e-6)
            gn = grads[i - 1].double()
            if freq is not None:
                p = pos.double()[:, None, :, None]
                gn = od.rotate(gn, -(p * freq), inter, amp)
            terms = (gn * xh).abs().sum((0, 1, 2))
            _check(dev_grads[i], gr[i], dtype, terms, name, units=64 + B * T * h)


def test_positions_of_one_row_and_none():
    """positions [T] and None (0 .. T - 1) give what the same positions [B, T] give."""
    from edifice_amd import fused_scan as fs
    announce("rotary_positions")
    case = (2, 9, 2, 1, 64, 64, False, True, 1.0, torch.float32)
    x, w, freq, _, _ = _make(case)
    args = (x.cuda(), 2, 1, freq.cuda())
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    kw = dict(q_weight=w[0].cuda(), k_weight=w[1].cuda())
    a = fs.split_heads_rotary(*args, **kw)
    b = fs.split_heads_rotary(*args, pos, **kw)
    c = fs.split_heads_rotary(*args, pos.expand(2, 9), **kw)
    for s, t, u in zip(a, b, c):
        assert torch.equal(s, t) and torch.equal(t, u)


def test_plain_split_is_the_block_split():
    """Without weights and frequencies the pass is fs.split_heads, and a misaligned x gives the same."""
    from edifice_amd import fused_scan as fs
    announce("rotary_plain_split")
    x = torch.randn(2, 5, 3 * 4 * 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    want = fs.split_heads(x, 3, 4)
    for o, r in zip(fs.split_heads_rotary(x, 4, 4), want):
        assert torch.equal(o, r)
    buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    buf[1:] = x.reshape(-1)
    for o, r in zip(fs.split_heads_rotary(buf[1:].view(x.shape), 4, 4), want):
        assert torch.equal(o, r)


def test_far_and_negative_positions():
    """Positions to 2^31 - 1 and negative ones: the angle is reduced in float64 (2^31 turns leave 2^-22 of one)."""
    from edifice_amd import fused_scan as fs
    announce("rotary_far")
    case = (1, 4, 2, 1, 64, 64, False, False, 1.0, torch.float32)
    x, w, freq, _, _ = _make(case)
    pos = torch.tensor([[-7, 0, 123456789, 2 ** 31 - 1]], dtype=torch.int32)
    out = fs.split_heads_rotary(x.cuda(), 2, 1, freq.cuda(), pos.cuda())
    ref = od.split_heads_rotary(x.double(), 2, 1, freq, pos)
    for o, r in zip(out[:2], ref[:2]):  # float64 products of 2^31 are off by up to 2^-22 turns: 1.5e-6 rad, 32 more units
        _check(o, r, torch.float32, 1.5 * r.abs().amax(-1, keepdim=True), "far", units=128)


def test_captured_and_replayed():
    """A captured forward replays on new contents of its inputs, eager work between the replays."""
    from edifice_amd import fused_scan as fs
    announce("rotary_graph")
    case = (2, 17, 4, 2, 64, 64, False, True, 1.0, torch.bfloat16)
    x, w, freq, pos, _ = _make(case)
    xs, ps = x.cuda(), pos.cuda()
    kw = dict(frequencies=freq.cuda(), q_weight=w[0].cuda(), k_weight=w[1].cuda())
    fs.split_heads_rotary(xs, 4, 2, positions=ps, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fs.split_heads_rotary(xs, 4, 2, positions=ps, **kw)
    for seed in range(1, 4):
        x2, _, _, p2, _ = _make(case, seed)
        xs.copy_(x2)
        ps.copy_(p2)
        want = fs.split_heads_rotary(xs, 4, 2, positions=ps, **kw)
        graph.replay()
        torch.cuda.synchronize()
        for o, r in zip(out, want):
            assert torch.equal(o, r)


def test_gradient_against_differences():
    """sum(g . out) along a direction, central differences of the float64 form against the kernel's gradients."""
    announce("rotary_differences")
    case = (1, 5, 2, 1, 32, 32, True, True, 1.1, torch.float32)
    B, T, Hq, Hkv, d, rot, inter, norm, amp, dtype = case
    x, w, freq, pos, grads = _make(case)
    _, g = _run(case, x, w, freq, pos, grads)
    gen = torch.Generator().manual_seed(9)
    dirs = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in (x, w[0], w[1])]

    def f(e):
        a, b, c = (t.double() + e * u for t, u in zip((x, w[0], w[1]), dirs))
        out = od.split_heads_rotary(a, Hq, Hkv, freq, pos, b, c, 1e-6, inter, amp)
        return sum((o * r.double()).sum() for o, r in zip(out, grads))

    want = float((f(1e-5) - f(-1e-5)) / 2e-5)
    got = sum(float((t.cpu().double() * u).sum()) for t, u in zip(g, dirs))
    size = sum(float((t.cpu().double() * u).abs().sum()) for t, u in zip(g, dirs))
    assert math.isfinite(got) and abs(got - want) <= 1e-5 * size
