"""The 8-bit paged cache without a GPU: what the C entry points and the Python ops refuse, and the oracle's own numbers."""
import math

import pytest
import torch

from edifice_amd import fused_scan as fs
from edifice_amd._native import EdificeHipError, lib
from oracle import decoder as od

P = 16  # a non-null address that no refused call reads


def _write(L, B=1, T=1, hkv=1, d=64, blocks=4, block=16, k=P, ks=P, vs=P, dtype=1, code=0):
    return L.edf_paged_cache_write8(None, k, P, P, P, P, ks, vs, B, T, hkv, d, blocks, block, dtype, code)


def _read(L, R=1, total=4, hkv=1, d=64, blocks=4, block=16, width=2, kc=P, ks=P, vs=P, dtype=1, code=0):
    return L.edf_paged_cache_read(None, kc, P, ks, vs, P, P, P, P, R, total, hkv, d, blocks, block, width, dtype, code)


def _attend(L, B=1, hq=2, hkv=1, d=64, blocks=4, block=16, width=2, window=0, sinks=0, q=P, ks=P, ws=None, wsb=0, dtype=1,
            code=0):
    return L.edf_paged_attention8(None, q, P, P, ks, P, P, P, P, ws, wsb, B, hq, hkv, d, blocks, block, width, window,
                                  sinks, dtype, code)


@pytest.mark.parametrize("call, code, message", [
    (lambda L: _write(L, T=0), 1, b"dimensions must be positive"),
    (lambda L: _write(L, dtype=2), 1, b"dtype"),
    (lambda L: _write(L, code=2), 1, b"code"),
    (lambda L: _write(L, code=-1), 1, b"code"),
    (lambda L: _write(L, k=None), 1, b"null"),
    (lambda L: _write(L, ks=None), 1, b"null"),
    (lambda L: _write(L, vs=None), 1, b"null"),
    (lambda L: _write(L, blocks=1 << 27), 2, b"2^31"),
    (lambda L: _write(L, block=1 << 20, d=256), 2, b"2^28"),
    (lambda L: _write(L, B=1 << 20, T=1 << 14, block=1), 2, b"too many"),
    (lambda L: _read(L, total=0), 1, b"dimensions must be positive"),
    (lambda L: _read(L, R=0), 1, b"dimensions must be positive"),
    (lambda L: _read(L, dtype=3), 1, b"dtype"),
    (lambda L: _read(L, code=5), 1, b"code"),
    (lambda L: _read(L, kc=None), 1, b"null"),
    (lambda L: _read(L, ks=None), 1, b"null"),
    (lambda L: _read(L, vs=None, code=1), 1, b"null"),
    (lambda L: _read(L, width=1 << 27), 2, b"2^31"),
    (lambda L: _read(L, total=1 << 31), 2, b"2^31"),
    (lambda L: _read(L, total=1 << 30, hkv=1 << 10), 2, b"too large"),
    (lambda L: _attend(L, width=0), 1, b"dimensions must be positive"),
    (lambda L: _attend(L, hq=3, hkv=2), 1, b"multiple"),
    (lambda L: _attend(L, code=7), 1, b"code"),
    (lambda L: _attend(L, ks=None), 1, b"null"),
    (lambda L: _attend(L, q=None), 1, b"null"),
    (lambda L: _attend(L, d=257), 2, b"head_dim"),
    (lambda L: _attend(L, window=-1), 1, b"window"),
    (lambda L: _attend(L, blocks=1 << 28), 2, b"2^31"),
    (lambda L: _attend(L, width=1 << 12), 4, b"workspace"),
])
def test_entry_points_refuse(call, code, message):
    L = lib()
    assert call(L) == code
    assert message in L.edf_last_error()


def test_workspace_query_of_refused_sizes():
    L = lib()
    assert L.edf_paged_attention8_workspace_bytes(1, 1, 2, 64, 4096, 16, 0, 0) == 0
    assert L.edf_paged_attention8_workspace_bytes(1, 2, 1, 64, 4096, 16, 0, 0) > 0


def _cache(blocks=2, hkv=1, block=4, d=8, dtype=torch.int8):
    return torch.zeros(blocks, hkv, block, d).to(dtype), torch.zeros(blocks, hkv)


I32 = torch.int32


@pytest.mark.parametrize("call, message", [
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c), "k_scale"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c, s), "v_scale"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c, s.double(), s), "k_scale"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c, s[:1], s), "k_scale"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c.to(torch.float8_e4m3fn), s, s), "dtype"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c.float(), c.float(), s, s), "scales belong"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c.to(torch.uint8), c, s, s), "scales belong"),
    (lambda k, c, s: fs.paged_cache_write(k.requires_grad_(), k, torch.zeros(1, 3, dtype=I32), c, c, s, s), "derivative"),
    (lambda k, c, s: fs.paged_cache_write(k, k, torch.zeros(1, 3, dtype=I32), c, c, s, s), "GPU tensors"),
    (lambda k, c, s: fs.paged_cache_write(k[..., :4], k[..., :4], torch.zeros(1, 3, dtype=I32), c, c, s, s), "must be"),
    (lambda k, c, s: fs.paged_cache_read(c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32), 3, s, s), "offsets"),
    (lambda k, c, s: fs.paged_cache_read(c, c, torch.zeros(1, 1), torch.zeros(2, dtype=I32), 3, s, s), "table"),
    (lambda k, c, s: fs.paged_cache_read(c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(2, dtype=I32), 3), "k_scale"),
    (lambda k, c, s: fs.paged_cache_read(c.float(), c.float(), torch.zeros(1, 1, dtype=I32), torch.zeros(2, dtype=I32), 3,
                                         dtype=torch.bfloat16), "as it is"),
    (lambda k, c, s: fs.paged_cache_read(c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(2, dtype=I32), 3, s, s),
     "GPU tensors"),
    (lambda k, c, s: fs.paged_attention(k[:, :, 0], c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32)),
     "k_scale"),
    (lambda k, c, s: fs.paged_attention(k[:, :, 0], c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32),
                                        k_scale=s, v_scale=s.t().contiguous()), "v_scale"),
    (lambda k, c, s: fs.paged_attention(k[:, :, 0], c, c, torch.zeros(1, 1, dtype=I32), torch.zeros(1, dtype=I32),
                                        k_scale=s, v_scale=s.requires_grad_()), "derivative"),
])
def test_python_refuses(call, message):
    c, s = _cache()
    with pytest.raises(EdificeHipError, match=message):
        call(torch.zeros(1, 1, 3, 8), c, s)


def test_oracle_numbers_are_the_types():
    """The oracle's rounding to e4m3 is torch's, on every value it can meet, and to int8 that of round() with ties to even."""
    g = torch.Generator().manual_seed(0)
    y = torch.cat([torch.randn(4000, generator=g) * 2.0 ** e for e in range(-14, 7)]).clamp(-448, 448)
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[torch.isfinite(every)].sort().values
    y = torch.cat([y, every, (every[1:] + every[:-1]) / 2])  # the numbers and the ties between them
    assert torch.equal(od.round_code(y.double(), "e4m3"), y.to(torch.float8_e4m3fn).double())
    z = torch.arange(-300, 301) / 2
    assert od.round_code(z.double(), "int8").tolist() == [max(-127, min(127, round(float(v)))) for v in z]


@pytest.mark.parametrize("code, top", [("int8", 127), ("e4m3", 448)])
def test_oracle_scale_is_the_least(code, top):
    for amax in [2.0 ** -90, 1e-9, 0.3, 1.0, 1.75, 1.7500001, 448.0, 449.0, 1e30]:
        s = od.least_scale(amax, code)
        assert amax / s <= top * (1 + 2.0 ** -22)
        assert amax / s > (top * (1 - 2.0 ** -22) if code == "int8" else top / 2)
    assert od.least_scale(0.0, code) == 0 and od.least_scale(1e-40, code) == 2.0 ** -100
    assert math.isnan(od.least_scale(math.inf, code)) and math.isnan(od.least_scale(math.nan, code))
