"""Attention over packed texts without a GPU: what the C entry points and the Python op refuse, and the oracle's pins."""
import math

import pytest
import torch

from edifice_amd import fused_scan as fs
from edifice_amd._native import EdificeHipError, lib
from oracle import decoder as od

P = 16  # a non-null address that no refused call reads


def _fwd(L, H=2, hkv=1, N=4, M=4, S=1, d=64, window=0, sinks=0, q=P, off=P, ws=None, wsb=0, dtype=1):
    return L.edf_packed_attention(None, q, P, P, off, P, P, None, ws, wsb, H, hkv, N, M, S, d, window, sinks, dtype)


def _bwd(L, H=2, hkv=1, N=4, M=4, S=1, d=64, lse=P, ws=P, wsb=1 << 40, window=0):
    return L.edf_packed_attention_backward(None, P, P, P, P, P, P, P, lse, P, P, P, ws, wsb, H, hkv, N, M, S, d, window, 0, 1)


@pytest.mark.parametrize("call, code, message", [
    (lambda L: _fwd(L, N=0), 1, b"dimensions must be positive"),
    (lambda L: _fwd(L, M=0), 1, b"dimensions must be positive"),
    (lambda L: _fwd(L, S=-1), 1, b"dimensions must be positive"),
    (lambda L: _fwd(L, H=3, hkv=2), 1, b"multiple"),
    (lambda L: _fwd(L, dtype=2), 1, b"dtype"),
    (lambda L: _fwd(L, window=-1), 1, b"window"),
    (lambda L: _fwd(L, sinks=-1), 1, b"window"),
    (lambda L: _fwd(L, d=129), 2, b"head_dim"),
    (lambda L: _fwd(L, N=1 << 30), 2, b"below"),
    (lambda L: _fwd(L, H=1 << 20, N=1 << 20), 2, b"too large"),
    (lambda L: _fwd(L, q=None), 1, b"null"),
    (lambda L: _fwd(L, off=None), 1, b"null"),
    (lambda L: _fwd(L, M=1 << 20), 4, b"workspace"),
    (lambda L: _bwd(L, lse=None), 1, b"lse"),
    (lambda L: _bwd(L, ws=None), 4, b"workspace"),
    (lambda L: _bwd(L, wsb=15), 4, b"workspace"),
    (lambda L: _bwd(L, d=200), 2, b"head_dim"),
    (lambda L: _bwd(L, window=-2), 1, b"window"),
])
def test_entry_points_refuse(call, code, message):
    L = lib()
    assert call(L) == code
    assert message in L.edf_last_error()


def test_workspace_query_of_refused_sizes():
    L = lib()
    assert L.edf_packed_attention_workspace_bytes(1, 2, 4, 4, 1, 64, 0, 0, 1) == 0
    assert L.edf_packed_attention_backward_workspace_bytes(1, 0, 4, 4, 1, 64, 0, 0, 1) == 0


def _q(h=2, n=4, d=8):
    return torch.zeros(h, n, d)


OFF = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("call, message", [
    (lambda: fs.packed_attention(_q(), _q(), _q(), OFF), "GPU tensors"),
    (lambda: fs.packed_attention(_q(), _q().bfloat16(), _q(), OFF), "dtype"),
    (lambda: fs.packed_attention(_q(3), _q(2), _q(2), OFF), "multiple"),
    (lambda: fs.packed_attention(_q(), _q(n=5), _q(n=5), OFF), "M = N"),
    (lambda: fs.packed_attention(_q(), _q(), _q(n=5), OFF), "needs"),
    (lambda: fs.packed_attention(_q(), _q(d=4), _q(d=4), OFF), "needs"),
    (lambda: fs.packed_attention(_q()[None].expand(2, 2, 4, 8), _q()[None], _q()[None], OFF), "rows, d"),
    (lambda: fs.packed_attention(_q()[None], _q(), _q(), OFF), "rows, d"),
    (lambda: fs.packed_attention(_q(), _q(), _q(), OFF.long()), "int32"),
    (lambda: fs.packed_attention(_q(), _q(), _q(), OFF[None]), "1-d"),
    (lambda: fs.packed_attention(_q(), _q(), _q(), OFF[:0]), "offsets"),
    (lambda: fs.packed_attention(_q(), _q(), _q(), OFF, OFF[:1]), "key_offsets"),
])
def test_python_refuses(call, message):
    with pytest.raises(EdificeHipError, match=message):
        call()


def test_oracle_is_windowed_attention_of_each_text():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(h, 12, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    for window, sinks in ((0, 0), (3, 1)):
        got = od.packed_attention(q, k, v, [0, 5, 5, 11], [0, 5, 5, 11], window, sinks)
        for a, b in ((0, 5), (5, 11)):
            want = od.window_attention(q[None, :, a:b], k[None, :, a:b], v[None, :, a:b], window or b - a, sinks)[0]
            assert torch.allclose(got[:, a:b], want, atol=1e-12)
        assert not got[:, 11:].any()
    # the last queries alone are the last rows; queries that come before every key answer with zeros
    whole = od.packed_attention(q, k, v, [0, 12], [0, 12], 5, 2)
    assert torch.allclose(od.packed_attention(q[:, 9:], k, v, [0, 3], [0, 12], 5, 2), whole[:, 9:], atol=1e-12)
    few = od.packed_attention(q, k[:, :4], v[:, :4], [0, 12], [0, 4])
    assert not few[:, :8].any() and bool(few[:, 8:].any())


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 5, 4, generator=g, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(1, 7, 4, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda *x: od.packed_attention(*x, [0, 2, 5], [0, 1, 7], 3, 1), (q, k, v))
    assert math.isfinite(float(q.detach().sum()))


def _cache(**opts):
    from edifice_amd import blocks
    m = blocks.build("gqa", embed_size=32, num_heads=4, num_kv_heads=2)
    return m, m.paged_cache(2, 12, block_size=4, **opts)


@pytest.mark.parametrize("lengths, taken, counts, room", [
    ([0, 0], 0, None, True),
    ([5, 0], 2, [7, 3], True),        # 12 tokens of three pages, and one page
    ([5, 0], 2, [8, 0], False),       # past the table's width
    ([5, 0], 5, [3, 0], True),        # within the page that is held
    ([5, 0], 5, [4, 4], False),       # two pages, one left
    ([5, 0], 2, [-9, 100], True),     # taken as 0 .. the tokens asked for
])
def test_room_for_several_tokens(lengths, taken, counts, room):
    _, c = _cache()
    c.lengths[:] = torch.tensor(lengths, dtype=torch.int32)
    for r, n in enumerate(lengths):
        c.table[r, :-(-n // 4)] = torch.arange(-(-n // 4), dtype=torch.int32)
    c.taken[0] = taken
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    assert c.has_room(12 if lengths == [0, 0] else 8, counts) == room
    c.lengths[1], c.table[1, 0] = 1, -1  # a token that found no page
    assert not c.has_room(1, None)


def test_go_on_refuses_before_anything_moves(monkeypatch):
    from edifice_amd import blocks
    monkeypatch.setattr(fs, "paged_extend", lambda *a: (_ for _ in ()).throw(AssertionError("made room")))
    m, c = _cache()
    with pytest.raises(ValueError, match="pages for all"):
        m.go_on(torch.zeros(2, 13, 32), c)
    with pytest.raises(ValueError, match="x must be"):
        m.go_on(torch.zeros(2, 3, 31), c)
    wide = blocks.build("gqa", embed_size=32, hidden_size=320, num_heads=2)
    for tokens in (1, 2):
        with pytest.raises(ValueError, match="head_dim"):
            wide.go_on(torch.zeros(2, tokens, 32), wide.paged_cache(2, 8))
    with pytest.raises(ValueError, match="rows, embed"):
        m.packed(torch.zeros(1, 4, 32), OFF)
    with pytest.raises(ValueError, match="attention blocks"):
        blocks.build("mamba", embed_size=32).packed(torch.zeros(4, 32), OFF)


def test_eight_bit_cache_of_a_model():
    m, c = _cache(dtype=torch.int8)
    assert c.k[0].dtype == torch.int8 and c.k_scale[0].shape == (6, 2) and c.k_scale[0].dtype == torch.float32
    assert _cache()[1].k_scale[0] is None
    with pytest.raises(EdificeHipError, match="GPU tensors"):
        m.step(torch.zeros(2, 1, 32), c)  # the cache fits the model; the ops take no CPU tensors
    with pytest.raises(ValueError, match="the cache holds"):
        m.step(torch.zeros(2, 1, 32), _cache(dtype=torch.bfloat16)[1])


@pytest.mark.parametrize("off", [OFF.long(), OFF[:0], OFF[None], OFF.to("meta")], ids=["int64", "empty", "2-d", "elsewhere"])
def test_packed_model_refuses_offsets(off):
    """Before they are looked up: an index past them would end the process on the GPU."""
    m, _ = _cache()
    with pytest.raises(ValueError, match="offsets must be"):
        m.packed(torch.zeros(4, 32), off)


def test_no_rows_and_no_places():
    m, _ = _cache()
    assert m.packed(torch.zeros(0, 32), OFF[:1]).shape == (0, m.final_norm.weight.numel())
    assert m.paged_cache(0, 12).has_room(3)


@pytest.mark.parametrize("sizes", [dict(N=1 << 29), dict(M=1 << 29), dict(sinks=1 << 29), dict(S=1 << 28)], ids=str)
def test_sizes_whose_sums_pass_an_int(sizes):
    L = lib()
    assert _fwd(L, **sizes) == 2 and b"below 2^29" in L.edf_last_error()


@pytest.mark.parametrize("opts", [{}, dict(dtype=torch.int8)], ids=["own type", "int8"])
def test_no_places_go_on(opts, monkeypatch):
    """No place: no states, and the cache is as it was."""
    m, _ = _cache()
    c = m.paged_cache(0, 12, block_size=4, **opts)
    none = torch.zeros(0, 3, dtype=torch.int32)
    monkeypatch.setattr(fs, "paged_extend", lambda *a: (none, none, torch.zeros(1, dtype=torch.int32)))
    for counts in (None, torch.zeros(0, dtype=torch.int32)):
        for method in (m.go_on, m.step):
            assert method(torch.zeros(0, 3, 32), c, counts).shape == (0, 3, m.final_norm.weight.numel())
    assert not c.lengths.numel() and int(c.taken) == 0
