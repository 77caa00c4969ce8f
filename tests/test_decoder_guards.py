"""What the decoder's attention operators and the paged cache do with calls that they refuse or cannot serve, without a
GPU: a refusal leaves the process and the cache as they were."""
import itertools

import pytest
import torch
from torch.autograd import forward_ad

from edifice_amd import blocks
from edifice_amd import fused_scan as fs
from edifice_amd._native import EdificeHipError, lib
from oracle import decoder as od

INT_MAX = 2 ** 31 - 1


@pytest.fixture
def host_tensors(monkeypatch):
    """CPU tensors pass for the current GPU's: a call reaches the entry point, which refuses before it launches."""
    monkeypatch.setattr(fs, "_here", lambda *ts: 0)


def test_workspace_query_of_any_sizes():
    """The size queries answer for every size an int holds (fewer query heads than key heads among them)."""
    L = lib()
    assert L.edf_paged_attention_workspace_bytes(1, 1, 2, 64, 4, 16, 0, 0) == 0
    assert L.edf_paged_attention_workspace_bytes(1, 3, 2, 64, 4096, 16, 0, 0) == 0
    for c in itertools.product((1, INT_MAX), (1, 2, INT_MAX), (1, 2, INT_MAX), (1, 257), (1, INT_MAX), (1, INT_MAX),
                               (0, 5, INT_MAX), (0, INT_MAX)):
        L.edf_paged_attention_workspace_bytes(*c)
    for c in itertools.product((1, INT_MAX), (1, 3, INT_MAX), (1, 2, INT_MAX), (1, INT_MAX), (1, 64, INT_MAX),
                               (1, INT_MAX), (0, INT_MAX), (0, 1)):
        L.edf_window_attention_backward_workspace_bytes(*c)


@pytest.mark.parametrize("heads, kv_heads", [(1, 2), (3, 2), (2, 4)])
def test_paged_attention_refuses_head_counts(host_tensors, heads, kv_heads):
    """Query heads that are no multiple of the cache's, fewer of them too, are refused with a message."""
    q, cache = torch.zeros(1, heads, 64), torch.zeros(2, kv_heads, 8, 64)
    with pytest.raises(EdificeHipError, match="multiple"):
        fs.paged_attention(q, cache, cache.clone(), torch.zeros(1, 2).int(), torch.ones(1).int())


def _listed(table, old, new, free, block, tokens, taken=None):
    """paged_extend on the CPU, by the oracle."""
    at = max(int(taken), 0) if taken is not None else 0
    t, slots, positions, used = od.paged_extend(table.tolist(), old.tolist(), new.tolist(), free.tolist()[at:], block,
                                                tokens)
    table.copy_(torch.tensor(t))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return i32(slots), i32(positions), i32([at + used])


def test_a_missing_page_is_reported_until_its_place_is_released(monkeypatch):
    """Another place's release gives pages back and takes no report away: the place's later tokens of the missing page
    find none, which the report says."""
    monkeypatch.setattr(fs, "paged_extend", _listed)
    c = blocks.PagedCache(1, 3, 8, 1, 32, block_size=4, num_blocks=1, device="cpu")
    counts = lambda *n: torch.tensor(n, dtype=torch.int32)  # noqa: E731
    c.extend(1, counts(1, 0, 0))
    assert not c.exhausted()
    c.extend(1, counts(0, 1, 0))
    assert c.exhausted() and c.table.tolist() == [[0, -1], [-1, -1], [-1, -1]]
    c.release(0)
    slots, _ = c.extend(3, counts(0, 3, 0))
    assert slots.tolist()[1] == [-1, -1, -1] and c.exhausted()
    c.extend(1, counts(0, 1, 0))  # the next page is found
    assert c.table.tolist()[1] == [-1, 0] and c.exhausted()
    c.release(1)
    assert not c.exhausted()
    assert c.extend(4, counts(4, 0, 0))[0].tolist()[0] == [0, 1, 2, 3] and not c.exhausted()
    c.release(0)
    c.lengths[2] = 9  # past the table's row
    assert c.exhausted()


def test_rotary_angles_serve_inference_and_training(monkeypatch):
    """The angles that a block keeps: float64 on its device from the start, fit for training whichever mode came first,
    and those of its present options."""
    seen = []
    monkeypatch.setattr(fs, "split_heads_rotary", lambda x, hq, hkv, f, *rest: seen.append(f))
    x = torch.zeros(1, 3, 32)
    with torch.inference_mode():
        a = blocks.GQAttention(32, 4, 2, rotary_dim=8, rotary_base=100.0)
        b = blocks.GQAttention(32, 4, 2, rotary_dim=8, rotary_base=100.0)
    for m in (a.bfloat16(), blocks.GQAttention(32, 4, 2, rotary_dim=8, rotary_base=100.0)):
        with torch.inference_mode():
            m._heads(x.to(m.q_proj.weight.dtype))
        want = fs.rotary_frequencies(8, 100.0, device="cpu")
        assert not seen[-1].is_inference() and torch.equal(seen[-1], want) and seen[-1].dtype == torch.float64
    b.rotary_base, b.rotary_dim = 50.0, 4
    b._heads(x)
    assert torch.equal(seen[-1], fs.rotary_frequencies(4, 50.0, device="cpu"))
    meta = blocks.GQAttention(32, 4, 2, rotary_dim=8).to("meta")
    assert meta._frequencies.device.type == "meta"
    assert torch.equal(meta.to_empty(device="cpu")._frequencies, fs.rotary_frequencies(8, device="cpu"))
    b.rotary_dim = 0
    b._heads(x)
    assert seen[-1] is None


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(host_tensors, monkeypatch, grad_mode):
    """A tangent on any input is refused, as by the other ops, and not dropped."""
    monkeypatch.setattr(fs.nat, "call", lambda *a: None)
    x, w = torch.zeros(1, 3, 4 * 32), torch.ones(32)
    q, k = torch.zeros(1, 4, 8, 64), torch.zeros(1, 2, 8, 64)
    cache, i32 = torch.zeros(2, 2, 8, 64), torch.zeros(1, 2).int()
    calls = [(lambda x, w: fs.split_heads_rotary(x, 2, 1, None, None, w, w), (x, w)),
             (lambda q, k, v: fs.window_attention(q, k, v, 4), (q, k, k)),
             (lambda q, k, v: fs.paged_attention(q, k, v, i32, i32[0, :1]), (q[:, :, 0], cache, cache)),
             (lambda k, v, kc, vc: fs.paged_cache_write(k, v, i32[:, :1], kc, vc), (k[:, :, :1], k[:, :, :1], cache, cache))]
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        for call, args in calls:
            call(*args)  # tensors without a tangent pass
            for i, t in enumerate(args):
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises((NotImplementedError, EdificeHipError)):
                    call(*args[:i], dual, *args[i + 1:])


def _state(c):
    return [t.clone() for t in (c.table, c.lengths, c.free, c.taken)]


def _unmoved(c, before):
    return all(torch.equal(a, b) for a, b in zip(_state(c), before))


def test_an_extension_that_raises_moves_nothing():
    """Refused arguments, and an op that raises (it takes no CPU tensors): lengths and pages stay."""
    c = blocks.PagedCache(1, 2, 8, 1, 32, block_size=4, device="cpu")
    c.lengths[0] = 3
    before = _state(c)
    for tokens, counts in ((0, None), (-1, None), (-2, torch.ones(2)), (1, torch.ones(3).int()), (1, torch.ones(2)),
                           (1, torch.ones(2, dtype=torch.int32))):
        with pytest.raises((ValueError, EdificeHipError)):
            c.extend(tokens, counts)
        assert _unmoved(c, before), (tokens, counts)


def _gqa(num_heads=4, **opts):
    return blocks.build("gqa", embed_size=32, num_heads=num_heads, num_kv_heads=2, window=4, **opts)


_MAMBA = lambda: blocks.build("mamba", embed_size=32)  # noqa: E731
_WIDE = lambda: blocks.build("gqa", embed_size=32, hidden_size=320, num_heads=2)  # noqa: E731


@pytest.mark.parametrize("model, owner, x, cache", [
    (_gqa, None, torch.zeros(2, 1, 31), {}),
    (_gqa, None, torch.zeros(2, 0, 32), {}),
    (_gqa, None, torch.zeros(2, 32), {}),
    (_gqa, None, torch.zeros(3, 1, 32), {}),
    (_gqa, None, torch.zeros(2, 1, 32, dtype=torch.bfloat16), {}),
    (_gqa, None, torch.zeros(2, 1, 32, device="meta"), {}),
    (_gqa, None, torch.zeros(2, 1, 32), dict(dtype=torch.bfloat16)),
    (_gqa, lambda: _gqa(num_layers=1), torch.zeros(2, 1, 32), {}),
    (_gqa, lambda: _gqa(num_heads=2), torch.zeros(2, 1, 32), {}),
    (_MAMBA, _gqa, torch.zeros(2, 1, 32), {}),
    (_WIDE, None, torch.zeros(2, 2, 32), {}),
], ids=["embed", "no tokens", "rank", "texts", "type", "device", "cache type", "layers", "head_dim", "family",
        "a prompt of wide heads"])
def test_a_step_that_does_not_fit_moves_nothing(monkeypatch, model, owner, x, cache):
    """A model, an input or a cache (here of the model ``owner``) that do not belong together: refused before the cache
    makes room."""
    monkeypatch.setattr(fs, "paged_extend", _listed)
    m = model()
    c = (owner() if owner else m).paged_cache(2, 8, **cache)
    before = _state(c)
    with pytest.raises(ValueError):
        m.step(x, c)
    assert _unmoved(c, before)


def test_a_prompt_into_a_long_place_is_refused(monkeypatch):
    """A place of 2^16 tokens and a prompt of as many: their product is zero in 32 bits."""
    monkeypatch.setattr(fs, "paged_extend", _listed)
    m = _gqa()
    c = m.paged_cache(2, 8)
    c.lengths[1] = 1 << 16
    for counts in (None, torch.tensor([0, 1 << 16], dtype=torch.int32)):
        with pytest.raises(ValueError, match="empty places"):
            m.step(torch.zeros(2, 2, 32), c, counts)
    assert c.lengths.tolist() == [0, 1 << 16]


def _uncalled(*a):
    raise AssertionError("an entry point was called")


def test_nothing_to_do(host_tensors, monkeypatch):
    """Batches of no texts and texts of no tokens answer with empty results, as the head split and the write do; other
    refusals stay."""
    monkeypatch.setattr(fs.nat, "call", _uncalled)
    z = lambda *s: torch.zeros(*s, requires_grad=True)  # noqa: E731
    for B, T in ((0, 5), (2, 0)):
        q, k, v = z(B, 4, T, 64), z(B, 2, T, 64), z(B, 2, T, 64)
        out = fs.window_attention(q, k, v, 3, 1)
        assert out.shape == q.shape
        assert [g.shape for g in torch.autograd.grad(out.sum(), (q, k, v))] == [t.shape for t in (q, k, v)]
        for window, sinks in ((0, 0), (2, -1)):
            with pytest.raises(EdificeHipError):
                fs.window_attention(q, k, v, window, sinks)
    cache, i32 = torch.zeros(2, 2, 8, 64), lambda *s: torch.zeros(*s, dtype=torch.int32)
    for shape in ((0, 4, 64), (0, 4, 1, 64)):
        assert fs.paged_attention(torch.zeros(shape), cache, cache, i32(0, 2), i32(0)).shape == shape
    with pytest.raises(EdificeHipError):
        fs.paged_attention(torch.zeros(0, 4, 64), cache, cache, i32(0, 2), i32(0), window=-1)
    for taken, used in ((None, 0), (torch.tensor([3], dtype=torch.int32), 3), (torch.tensor([-1], dtype=torch.int32), 0)):
        slots, positions, got = fs.paged_extend(i32(0, 2), i32(0), i32(0), i32(3), 8, 5, taken)
        assert slots.shape == positions.shape == (0, 5) and got.tolist() == [used] and got is not taken
    with pytest.raises(EdificeHipError):
        fs.paged_extend(i32(0, 2), i32(0), i32(0), i32(3), 8, 0)
