"""GPU parity: the rotary head split's backward where a workgroup takes several tiles of tokens in turn (sines rebuilt
behind a barrier, weight gradients carried over): calls of more than 1024 tiles.

Tolerances as in test_gpu_rotary.py, but for the weight gradients, whose terms (64 units of 2^-24 each) go through at
most 320 additions one after another: under 32 rows of a thread, up to 256 threads of an element in a workgroup (one
after another), 1024 workgroups in 64 columns of 16, and 16 + 2 joins of the columns."""
import pytest
import torch

from oracle import decoder as od
from tests.gpu_util import announce
from tests.test_gpu_rotary import _check, _double, _make, _run

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32

CASES = [
    # (B, T, Hq, Hkv, d, rot, interleaved, norm, amplitude, dtype); tiles of 2, 2, 1 and 2 tokens
    (1, 3001, 12, 2, 128, 128, False, True, 1.0, bf16),
    (2, 1777, 6, 1, 96, 48, True, True, 1.2, f32),
    (1, 1500, 2, 1, 255, 254, False, True, 0.7, bf16),
    (1, 2100, 12, 2, 128, 64, False, False, 1.0, bf16),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward_over_several_tiles(case):
    B, T, Hq, Hkv, d, rot, inter, norm, amp, dtype = case
    announce("split_heads_rotary tiles", case=case)
    x, w, freq, pos, grads = _make(case)
    _, got = _run(case, x, w, freq, pos, grads)
    leaves = [_double(x), _double(w[0]), _double(w[1])]
    ref = od.split_heads_rotary(leaves[0], Hq, Hkv, freq, pos, leaves[1], leaves[2], 1e-6, inter, amp)
    want = torch.autograd.grad(ref, [t for t in leaves if t is not None], [t.double() for t in grads])
    row = want[0].view(B, T, -1, d).abs().amax(-1, keepdim=True).expand(B, T, -1, d).reshape(want[0].shape)
    _check(got[0], want[0], dtype, 4 * row + 1e-3, "dx")
    if not norm:
        return
    for i, name, h, at in ((1, "dwq", Hq, 0), (2, "dwk", Hkv, Hq)):
        u = x.double().view(B, T, -1, d)[:, :, at:at + h].transpose(1, 2)
        xh = u / torch.sqrt(u.square().mean(-1, keepdim=True) + 1e-6)
        gn = od.rotate(grads[i - 1].double(), -(pos.double()[:, None, :, None] * freq), inter, amp)
        _check(got[i], want[i], dtype, (gn * xh).abs().sum((0, 1, 2)), name, units=64 + 320)
