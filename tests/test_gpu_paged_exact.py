"""GPU parity: attention over pages in bf16 is off by the rounding of its result and float32 sums alone.

Tolerance, per element: the probabilities go through the matrix product in two bf16 parts, off by 2^-16 of themselves
(each part's rounding is half a step, 2^-8 of what it rounds); 256 units of 2^-24 for the float32 sums and the
exponential; both of sum P |V|; half a step of bf16 of the result, 2^-8."""
import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce
from tests.test_gpu_paged import U, _pool

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


@pytest.mark.parametrize("case", [
    # lengths, Hq, Hkv, d, block, window, sinks
    ((700, 129, 128, 127), 8, 1, 64, 32, 0, 0),
    ((1000, 3, 260), 6, 2, 128, 64, 100, 4),
    ((300, 50), 40, 2, 128, 16, 0, 0),
    ((90, 41), 3, 1, 7, 4, 0, 0),
    ((130, 77), 4, 2, 256, 16, 0, 0),
    ((3000,), 2, 1, 256, 16, 0, 0),
    ((5000,), 2, 1, 128, 16, 0, 0),
], ids=str)
def test_probabilities_in_two_parts(case):
    from edifice_amd import fused_scan as fs
    lengths, Hq, Hkv, d, block, window, sinks = case
    announce("paged_exact", case=case)
    kc, vc, table, n, g = _pool(lengths, Hkv, d, block, bf16)
    vc = vc.abs()  # sums that do not cancel: a rounded P would show beside the result's own rounding
    q = torch.randn(len(lengths), Hq, d, generator=g).to(bf16)
    got = fs.paged_attention(*(t.cuda() for t in (q, kc, vc, table, n)), window=window, sinks=sinks).cpu().double()
    want, mag = od.paged_attention(q.double(), kc.double(), vc.double(), table, n, window, sinks)
    tol = (2.0 ** -16 + 256 * U) * mag + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_weights_of_a_row_add_to_one(d):
    """Values of one: the probabilities as the product has them add to the sum that divides.  All but the first key's
    are 0.50176, which one bf16 part would hold as 0.5, and 32 of them as 0.9967 of the row."""
    from edifice_amd import fused_scan as fs
    announce("paged_weights", d=d)
    score = -0.689637 * d ** 0.5 / 8  # log of 0.50176
    q, kc = torch.zeros(1, 2, d, dtype=bf16, device="cuda"), torch.zeros(2, 1, 16, d, dtype=bf16, device="cuda")
    q[..., :2] = 8.0
    kc[..., 0] = score
    kc[..., 1] = score - float(kc[0, 0, 0, 0])
    kc[0, 0, 0] = 0.0
    i32 = dict(dtype=torch.int32, device="cuda")
    got = fs.paged_attention(q, kc, torch.ones_like(kc), torch.tensor([[0, 1]], **i32), torch.tensor([32], **i32))
    assert torch.equal(got, torch.ones_like(got))
