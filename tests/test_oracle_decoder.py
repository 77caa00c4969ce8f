"""Pins of oracle/decoder.py (CPU): closed forms, the flash-attention oracle, finite differences."""
import math

import numpy as np
import pytest
import torch

from oracle import decoder as od
from oracle import scans


def _rand(*shape, seed=0):
    return torch.randn(*shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))


def test_window_over_the_whole_sequence_is_causal_attention():
    q, k, v = (_rand(2, 3, 17, 8, seed=s) for s in range(3))
    want = torch.from_numpy(scans.flash_attention(q.numpy(), k.numpy(), v.numpy(), True))
    assert torch.allclose(od.window_attention(q, k, v, 17), want, atol=1e-12)
    assert torch.allclose(od.window_attention(q, k, v, 1, 17), want, atol=1e-12)  # every key a sink


def test_window_of_one_returns_the_own_value():
    q, k, v = (_rand(1, 4, 9, 8, seed=s)[:, :n] for s, n in ((0, 4), (1, 2), (2, 2)))
    assert torch.equal(od.window_attention(q, k, v, 1), v.repeat_interleave(2, 1))


@pytest.mark.parametrize("T, window, sinks", [(9, 3, 2), (6, 10, 1), (7, 2, 0), (8, 3, 5)])
def test_window_mask_is_the_definition(T, window, sinks):
    m = od.window_mask(T, window, sinks)
    for i in range(T):
        for j in range(T):
            assert bool(m[i, j]) == (j <= i and (i - j < window or j < sinks))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_depends_on_the_distance_alone_and_keeps_lengths(interleaved):
    freq = 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    q, k = _rand(1, 8), _rand(1, 8, seed=1)
    turn = lambda u, p: od.rotate(u, p * freq[None], interleaved, 1.0)  # noqa: E731
    near, far = ((turn(q, p + 5) * turn(k, p)).sum() for p in (0, 123456))
    assert abs(near - far) < 1e-9
    assert abs(turn(q, 77.0).norm() - q.norm()) < 1e-12
    assert torch.equal(turn(q, 0.0), q)


def test_norm_gives_unit_mean_square():
    q, k, v = od.split_heads_rotary(_rand(1, 3, 4 * 6), 2, 1, wq=torch.ones(6).double(), wk=torch.ones(6).double(), eps=0)
    assert torch.allclose(q.square().mean(-1), torch.ones(1, 2, 3).double())


def test_gradients_against_finite_differences():
    q, k, v = (_rand(1, h, 6, 4, seed=s).requires_grad_() for s, h in ((0, 4), (1, 2), (2, 2)))
    assert torch.autograd.gradcheck(lambda *a: od.window_attention(*a, 3, 1), (q, k, v))
    x, w = _rand(1, 3, 4 * 6).requires_grad_(), (1 + 0.1 * _rand(6)).requires_grad_()
    freq = torch.tensor([1.0, 0.3], dtype=torch.float64)
    assert torch.autograd.gradcheck(
        lambda x, w: od.split_heads_rotary(x, 2, 1, freq, torch.tensor([3, 1, 9]), w, 2 * w, 1e-6, True, 1.2), (x, w))


def test_paged_attention_over_pages_in_order_is_attention():
    q, k, v = _rand(2, 4, 8), _rand(2, 2, 12, 8, seed=1), _rand(2, 2, 12, 8, seed=2)
    kc, vc = (t.view(2, 2, 3, 4, 8).permute(0, 2, 1, 3, 4).reshape(6, 2, 4, 8) for t in (k, v))
    table = torch.tensor([[0, 1, 2], [3, 4, 5]])
    got, mag = od.paged_attention(q, kc, vc, table, torch.tensor([12, 7]))
    for b, n in ((0, 12), (1, 7)):
        p = torch.softmax(q[b] @ k[b].repeat_interleave(2, 0)[:, :n].transpose(-1, -2) / math.sqrt(8), -1)
        want = torch.stack([p[h, h] @ v[b, h // 2, :n] for h in range(4)])
        assert torch.allclose(got[b], want) and bool((mag[b] >= got[b].abs() - 1e-12).all())


def test_paged_extend_by_hand():
    table, slots, pos, used = od.paged_extend([[7, -1, -1], [-1, -1, -1], [5, -1, -1]], [3, 0, 2], [6, 4, 2], [9, 8, 6],
                                              4, 3)
    assert table == [[7, 9, -1], [8, -1, -1], [5, -1, -1]] and used == 2
    assert slots == [[31, 36, 37], [32, 33, 34], [-1, -1, -1]]
    assert pos == [[3, 4, 5], [0, 1, 2], [-1, -1, -1]]
    # a list that is too short, and a table that is too narrow
    table, slots, _, used = od.paged_extend([[-1], [-1]], [0, 0], [6, 3], [2], 4, 6)
    assert table == [[2], [-1]] and used == 2
    assert slots == [[8, 9, 10, 11, -1, -1], [-1] * 6]
    assert np.array(slots).shape == (2, 6)
