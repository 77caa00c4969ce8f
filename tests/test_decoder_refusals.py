"""Refusals of the decoder's attention operators, without a GPU: the C entry points check before they launch, and the
Python ops raise on shapes, types and CPU tensors."""
import math

import pytest
import torch

from edifice_amd import fused_scan as fs
from edifice_amd._native import EdificeHipError, lib

P = 16  # a non-null address that no refused call reads


def _rotary(L, B=1, T=4, hq=2, hkv=1, d=64, rot=64, x=P, freq=P, wq=None, wk=None, dtype=1):
    return L.edf_heads_split_rotary(None, x, freq, None, wq, wk, P, P, P, B, T, hq, hkv, d, rot, 0, 0, 1e-6, 1.0, dtype)


def _window(L, B=1, hq=2, hkv=1, T=4, d=64, window=2, sinks=0, q=P, dtype=1):
    return L.edf_window_attention(None, q, P, P, P, None, B, hq, hkv, T, d, window, sinks, dtype)


def _window_bwd(L, lse=P, ws=P, wsb=1 << 30, window=2):
    return L.edf_window_attention_backward(None, P, P, P, P, P, lse, P, P, P, ws, wsb, 1, 2, 1, 4, 64, window, 0, 1)


def _paged(L, B=1, hq=2, hkv=1, d=64, blocks=4, block=16, width=2, window=0, sinks=0, q=P, ws=None, wsb=0, dtype=1):
    return L.edf_paged_attention(None, q, P, P, P, P, P, ws, wsb, B, hq, hkv, d, blocks, block, width, window, sinks, dtype)


def _extend(L, R=2, width=2, free=2, block=16, tokens=1, table=P, taken=None, used=P):
    return L.edf_paged_extend(None, table, P, P, P, taken, P, P, used, R, width, free, block, tokens)


def _write(L, B=1, T=1, hkv=1, d=64, blocks=4, block=16, k=P, dtype=1):
    return L.edf_paged_cache_write(None, k, P, P, P, P, B, T, hkv, d, blocks, block, dtype)


@pytest.mark.parametrize("call, code, message", [
    (lambda L: _rotary(L, T=0), 1, b"dimensions must be positive"),
    (lambda L: _rotary(L, dtype=2), 1, b"dtype"),
    (lambda L: _rotary(L, d=257, rot=0), 2, b"head_dim"),
    (lambda L: _rotary(L, rot=33), 1, b"rotary_dim"),
    (lambda L: _rotary(L, rot=66), 1, b"rotary_dim"),
    (lambda L: _rotary(L, rot=-2), 1, b"rotary_dim"),
    (lambda L: _rotary(L, freq=None), 1, b"null"),
    (lambda L: _rotary(L, x=None), 1, b"null"),
    (lambda L: _rotary(L, wq=P), 1, b"together"),
    (lambda L: _rotary(L, B=1 << 20, T=1 << 12), 2, b"2^31"),
    (lambda L: L.edf_heads_split_rotary_backward(None, P, P, None, P, P, P, P, P, P, P, P, None, 0, 1, 4, 2, 1, 64, 64, 0,
                                                 0, 1e-6, 1.0, 1), 4, b"workspace"),
    (lambda L: _window(L, T=0), 1, b"dimensions must be positive"),
    (lambda L: _window(L, hq=3, hkv=2), 1, b"multiple"),
    (lambda L: _window(L, window=0), 1, b"window"),
    (lambda L: _window(L, sinks=-1), 1, b"sinks"),
    (lambda L: _window(L, d=129), 2, b"head_dim"),
    (lambda L: _window(L, B=1 << 16, hq=1 << 15), 2, b"too large"),
    (lambda L: _window(L, B=1 << 10, T=1 << 27), 2, b"too large"),
    (lambda L: _window(L, sinks=(1 << 22) + 1), 2, b"sinks"),
    (lambda L: _window(L, q=None), 1, b"null"),
    (lambda L: _window(L, dtype=3), 1, b"dtype"),
    (lambda L: _window_bwd(L, lse=None), 1, b"lse"),
    (lambda L: _window_bwd(L, wsb=15), 4, b"workspace"),
    (lambda L: _window_bwd(L, ws=None), 4, b"workspace"),
    (lambda L: _window_bwd(L, window=-1), 1, b"window"),
    (lambda L: _paged(L, width=0), 1, b"dimensions must be positive"),
    (lambda L: _paged(L, hq=3, hkv=2), 1, b"multiple"),
    (lambda L: _paged(L, d=257), 2, b"head_dim"),
    (lambda L: _paged(L, window=-1), 1, b"window"),
    (lambda L: _paged(L, blocks=1 << 28), 2, b"2^31"),
    (lambda L: _paged(L, width=1 << 26), 2, b"2^30"),
    (lambda L: _paged(L, width=1 << 12), 4, b"workspace"),
    (lambda L: _paged(L, q=None), 1, b"null"),
    (lambda L: _extend(L, tokens=0), 1, b"dimensions must be positive"),
    (lambda L: _extend(L, R=1 << 20, tokens=1 << 11), 2, b"2^31"),
    (lambda L: _extend(L, table=None), 1, b"null"),
    (lambda L: _extend(L, taken=P, used=P), 1, b"two places"),
    (lambda L: _write(L, block=0), 1, b"dimensions must be positive"),
    (lambda L: _write(L, blocks=1 << 27), 2, b"2^31"),
    (lambda L: _write(L, B=1 << 20, T=1 << 10), 2, b"too many"),
    (lambda L: _write(L, k=None), 1, b"null"),
    (lambda L: _write(L, dtype=-1), 1, b"dtype"),
])
def test_entry_points_refuse(call, code, message):
    L = lib()
    assert call(L) == code and message in L.edf_last_error()


def test_workspace_queries():
    L = lib()
    assert L.edf_window_attention_backward_workspace_bytes(0, 1, 1, 1, 1, 1, 0, 1) == 0
    assert L.edf_paged_attention_workspace_bytes(1, 1, 1, 64, 0, 16, 0, 0) == 0
    rows = 2 * 8 * 4096 * 4
    assert L.edf_window_attention_backward_workspace_bytes(2, 8, 2, 4096, 128, 1024, 4, 1) >= rows
    # a table that one workgroup a head covers needs none, a long one does
    assert L.edf_paged_attention_workspace_bytes(1, 8, 8, 128, 1, 16, 0, 0) == 0
    assert L.edf_paged_attention_workspace_bytes(1, 8, 8, 128, 8192, 16, 0, 0) > 0


CPU = dict(q=(1, 4, 8, 64), k=(1, 2, 8, 64))


@pytest.mark.parametrize("call", [
    lambda t: fs.split_heads_rotary(t(1, 3, 256), 2, 1),
    lambda t: fs.split_heads_rotary(t(1, 3, 255), 2, 1),
    lambda t: fs.split_heads_rotary(t(3, 256), 2, 1),
    lambda t: fs.split_heads_rotary(t(1, 3, 256), 0, 1),
    lambda t: fs.split_heads_rotary(t(1, 3, 256), 2, 1, q_weight=t(64)),
    lambda t: fs.window_attention(t(*CPU["q"]), t(*CPU["k"]), t(*CPU["k"]), 4),
    lambda t: fs.paged_attention(t(1, 4, 64), t(2, 2, 8, 64), t(2, 2, 8, 64), t(1, 2).int(), t(1).int()),
    lambda t: fs.paged_cache_write(t(1, 2, 1, 64), t(1, 2, 1, 64), t(1, 1).int(), t(2, 2, 8, 64), t(2, 2, 8, 64)),
    lambda t: fs.paged_extend(t(2, 2).int(), t(2).int(), t(2).int(), t(3).int(), 16, 1),
    lambda t: fs.paged_extend(t(2, 2), t(2).int(), t(2).int(), t(3).int(), 16, 1),
    lambda t: fs.paged_attention(t(1, 4, 64).requires_grad_(), t(2, 2, 8, 64), t(2, 2, 8, 64), t(1, 2).int(), t(1).int()),
    lambda t: fs.paged_cache_write(t(1, 2, 1, 64).requires_grad_(), t(1, 2, 1, 64), t(1, 1).int(), t(2, 2, 8, 64),
                                   t(2, 2, 8, 64)),
])
def test_python_ops_refuse(call):
    with pytest.raises(EdificeHipError):
        call(lambda *s: torch.zeros(*s))


def test_rotary_frequencies():
    f = lambda **k: fs.rotary_frequencies(8, 100.0, device="cpu", **k)  # noqa: E731
    plain = torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64)
    assert torch.allclose(f(), plain, atol=1e-15) and f().dtype == torch.float64
    assert torch.allclose(f(scaling="linear", factor=4.0), plain / 4)
    based = f(scaling="base", factor=4.0)
    assert based[0] == 1 and torch.isclose(based[-1], plain[-1] / 4)
    parts = f(scaling="parts", factor=4.0, original_length=100, slow=1.0, fast=8.0)
    turns = 100 * plain / (2 * math.pi)  # 15.9, 5.03, 1.59, 0.50
    keep = ((turns - 1) / 7).clamp(0, 1)
    assert torch.allclose(parts, plain / 4 * (1 - keep) + plain * keep) and parts[0] == 1 and parts[3] == plain[3] / 4
    assert fs.rotary_frequencies(0, device="cpu").numel() == 0
    for bad in (dict(rotary_dim=3), dict(rotary_dim=4, base=0.0), dict(rotary_dim=4, scaling="other"),
                dict(rotary_dim=4, scaling="parts"), dict(rotary_dim=4, scaling="linear", factor=0.0)):
        with pytest.raises(EdificeHipError):
            fs.rotary_frequencies(**{"device": "cpu", **bad})


def test_build_refuses_attention_options_elsewhere():
    from edifice_amd import blocks
    with pytest.raises(TypeError):
        blocks.build("mamba", embed_size=32, window=4)
    with pytest.raises(ValueError):
        blocks.build("mamba", embed_size=32).paged_cache(1, 8)
    m = blocks.build("gqa", embed_size=32, num_heads=4, num_kv_heads=2, rotary_dim=8, qk_norm=True)
    assert tuple(m.state_dict()["blocks.1.attn.q_norm"].shape) == (8,)
