"""GPU parity: windowed attention in the tiles that every query of a block sees whole, and with scores that grow or fall
along the keys, so that the running maximum moves, stays behind and is passed, in every kernel.

Tolerances, per element, from arithmetic (h: half a step of the type, 0 for float32 inside; U = 2^-24):
  a score of terms of size s = scale sum |q||k| is off by at most (d + 8) U s (d additions, the scaling, the
    exponential's argument, as a power of two up to 1.45 s), and so is the logarithm of the row's sum: P by
    a = 3 (d + 8) U s of itself, s the row's largest;
  O  = sum P V / sum P: P is rounded in the product and in the sum: e_O = (2 h + 2 a + 256 U) sum P |V| + h |O|;
  the backward's P = exp(score - lse), lse of the rounded sum: off by b = h + 2 a of itself;
  dV = sum P dO, P rounded once more: (h + b + 256 U) sum P |dO| + h |dV|;
  dS = P (dP - D), D = sum dO O of the O that the forward left: e = P sum |dO| e_O + (h + b) |dS| + 256 U P (sum |dO||V|
    + sum |dO O|), so dQ: scale sum e |K| + h |dQ|, dK: scale sum e |Q| + h |dK|;
  probabilities below 2^-126 may be taken as zeros: less than 2^-100 in any of these sums of at most 2^20 terms."""
import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce
from tests.test_gpu_window_attention import H, U, _make, _within

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32


def _expected(case, q, k, v, do):
    """(value, tolerance) of O, dQ, dK, dV."""
    B, Hq, Hkv, T, d, window, sinks, dtype = case
    G, h, s = Hq // Hkv, H[dtype], d ** -0.5
    q, k, v, do = (t.double() for t in (q, k, v, do))
    kr, vr = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    p = od.window_probabilities(q, k, window, sinks)
    size = (q.abs() @ kr.abs().transpose(-1, -2)).masked_fill(~od.window_mask(T, window, sinks), 0.0)
    a = 3 * (d + 8) * U * s * size.amax(-1, keepdim=True)
    del size
    o = p @ vr
    eo = (2 * h + 2 * a + 256 * U) * (p @ vr.abs()) + max(h, U) * o.abs()
    ds = p * (do @ vr.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    b = h + 2 * a
    e = p * (do.abs() * eo).sum(-1, keepdim=True) + (h + b) * ds.abs()
    e += 256 * U * p * (do.abs() @ vr.abs().transpose(-1, -2) + (do * o).abs().sum(-1, keepdim=True))
    shared = lambda t: t.view(B, Hkv, G, T, d).sum(2)  # noqa: E731
    want = {"O": o, "dQ": s * ds @ kr, "dK": s * shared(ds.transpose(-1, -2) @ q), "dV": shared(p.transpose(-1, -2) @ do)}
    tol = {"dQ": s * e @ kr.abs(), "dK": s * shared(e.transpose(-1, -2) @ q.abs()),
           "dV": shared(((h + b + 256 * U) * p).transpose(-1, -2) @ do.abs())}
    return {n: (want[n], 2.0 ** -100 + (eo if n == "O" else tol[n] + max(h, U) * want[n].abs())) for n in want}


def _compare(case, q, k, v, do, off=0):
    from edifice_amd import fused_scan as fs
    window, sinks = case[5:7]

    def dev(t):  # ``off`` elements off 16 bytes
        buf = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
        buf[off:] = t.reshape(-1)
        return buf[off:].view(t.shape)
    leaves = [dev(t).requires_grad_() for t in (q, k, v)]
    out = fs.window_attention(*leaves, window, sinks)
    grads = torch.autograd.grad(out, leaves, dev(do))
    exp = _expected(case, q, k, v, do)
    for name, got in zip(("O", "dQ", "dK", "dV"), (out, *grads)):
        _within(got, *exp[name], name)


def _whole_tiles(T, window, sinks, block, keys):
    """Tiles of ``keys`` keys that all queries of a full block of ``block`` see, counted from the definition."""
    return sum(bool(od.window_mask(T, window, sinks)[q0:q0 + block, k0:k0 + keys].all())
               for q0 in range(0, T - block + 1, block) for k0 in range(sinks, T - keys + 1) if k0 % keys == 0)


WHOLE = [
    # (B, Hq, Hkv, T, d, window, sinks, dtype): grids of 160 blocks of 128 queries and more
    (2, 16, 4, 700, 128, 300, 5, bf16),
    (4, 8, 2, 700, 128, 1000, 0, bf16),
    (4, 8, 2, 650, 96, 400, 3, bf16),
    (4, 8, 4, 650, 80, 300, 0, bf16),
    (4, 8, 8, 650, 64, 333, 70, bf16),
    (4, 8, 2, 700, 32, 300, 1, bf16),
    (4, 8, 2, 700, 128, 300, 2, f32),
    (4, 8, 4, 650, 72, 300, 0, f32),
    (4, 8, 2, 650, 64, 1000, 0, f32),
    (4, 8, 2, 700, 32, 260, 40, f32),
]


@pytest.mark.parametrize("case", WHOLE, ids=str)
def test_whole_tiles(case):
    """The unmasked loops of the wide kernels, each width and type."""
    announce("window_whole", case=case)
    assert _whole_tiles(*case[3:4], *case[5:7], 128, 64 if case[7] == bf16 else 32) > 0
    _compare(case, *_make(case))


@pytest.mark.parametrize("case", [(1, 4, 2, 600, 128, 300, 2, bf16), (1, 2, 1, 600, 64, 600, 0, bf16),
                                  (1, 4, 1, 500, 90, 250, 3, bf16), (1, 4, 2, 600, 128, 300, 2, f32),
                                  (1, 2, 1, 500, 31, 500, 0, f32)], ids=str)
def test_whole_tiles_off_16_bytes(case):
    """The same loops where rows are read by elements."""
    announce("window_whole_off", case=case)
    assert _whole_tiles(*case[3:4], *case[5:7], 128, 64 if case[7] == bf16 else 32) > 0
    _compare(case, *_make(case), off=1)


@pytest.mark.parametrize("course", ["growing", "falling", "a step"])
@pytest.mark.parametrize("case", [
    (4, 8, 2, 700, 128, 400, 3, bf16), (4, 8, 2, 700, 128, 700, 0, bf16), (4, 8, 4, 650, 64, 400, 70, bf16),
    (4, 8, 2, 650, 96, 500, 0, bf16), (4, 8, 2, 700, 128, 400, 3, f32), (4, 8, 2, 650, 64, 650, 0, f32),
    (1, 4, 2, 400, 64, 300, 2, bf16), (1, 4, 2, 400, 128, 300, 0, f32)], ids=str)
def test_scores_that_move_the_maximum(case, course):
    """Keys that grow from 1 to 12 times their size along the text, that fall, or that are larger by a fifth from the
    middle on (scores past the running maximum by less than the factor at which it moves)."""
    announce("window_scores", case=case, course=course)
    q, k, v, do = _make(case)
    at = torch.linspace(0, 1, case[3], dtype=torch.float64)[:, None]
    size = {"growing": 1 + 11 * at, "falling": 12 - 11 * at, "a step": 3.0 + 0.6 * (at > 0.5)}[course]
    _compare(case, q, (k.double() * size).to(k.dtype), v, do)


@pytest.mark.parametrize("B, Hq, d", [(1, 2, 64), (1, 2, 128), (20, 8, 64), (20, 8, 96), (20, 8, 128)])
def test_the_weights_of_a_row_add_to_one(B, Hq, d):
    """Values of one: the sum that divides is that of the probabilities as the product has them, in the kernels of
    small and of large calls alike.  All but the first key's scores give 0.50176, which bf16 rounds to 0.5: divided by
    the unrounded sum, a row of 32 keys would answer 0.9967, which rounds to 0.99609."""
    from edifice_amd import fused_scan as fs
    announce("window_weights", B=B, d=d)
    T, score = 32, -0.689637 * d ** 0.5 / 8  # log of 0.50176
    q, k = (torch.zeros(B, Hq, T, d, dtype=bf16, device="cuda") for _ in range(2))
    q[..., :2] = 8.0
    k[..., 1:, 0] = score
    k[..., 1:, 1] = score - float(k[0, 0, 1, 0])
    assert torch.equal(fs.window_attention(q, k, torch.ones_like(q), T), torch.ones_like(q))
