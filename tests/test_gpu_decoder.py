"""The decoder's attention operators run together, as a model uses them: training through the block, and prompts and
steps over a paged cache, against float64 and against the whole sequence at once."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import decoder as od
from tests.conftest import assert_close
from tests.gpu_util import announce, host

pytestmark = pytest.mark.gpu

OPTS = dict(rotary_dim=16, qk_norm=True, window=9, sinks=2)


def _model(dtype, num_kv_heads=2, **opts):
    from edifice_amd import blocks
    torch.manual_seed(3)
    m = blocks.build("gqa", embed_size=48, hidden_size=96, num_heads=4, num_kv_heads=num_kv_heads, **opts)
    with torch.no_grad():
        for b in m.blocks:
            if b.attn.q_norm is not None:
                b.attn.q_norm.add_(0.3 * torch.randn(24))
                b.attn.k_norm.add_(0.3 * torch.randn(24))
    return m.to(device="cuda", dtype=dtype)


def _reference(w, x, nh, nkv, opts):
    """The model in float64 from its definition (torch, CPU), differentiable."""
    d = w["blocks.0.attn.q_proj.weight"].shape[0] // nh
    rot = opts.get("rotary_dim", 0)
    freq = opts.get("rotary_base", 10000.0) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot) if rot else None
    h = F.linear(x, w["input_projection.weight"], w["input_projection.bias"])
    for i in range(2):
        p = lambda s: w[f"blocks.{i}.{s}"]  # noqa: E731
        lin = lambda t, s: F.linear(t, p(s + ".weight"), p(s + ".bias"))  # noqa: E731
        ln = lambda t, s: F.layer_norm(t, (t.shape[-1],), p(s + ".weight"), p(s + ".bias"), 1e-5)  # noqa: E731
        n = ln(h, "attn_norm")
        qkv = torch.cat([lin(n, f"attn.{c}_proj") for c in "qkv"], -1)
        norm = [w.get(f"blocks.{i}.attn.{c}_norm") for c in "qk"]
        q, k, v = od.split_heads_rotary(qkv, nh, nkv, freq, None, *norm)
        o = od.window_attention(q, k, v, opts.get("window") or x.shape[1], opts.get("sinks", 0))
        h = h + lin(o.transpose(1, 2).reshape(h.shape[:2] + (nh * d,)), "attn.out_proj")
        h = h + lin(F.gelu(lin(ln(h, "ffn_norm"), "ffn_up")), "ffn_down")
    return F.layer_norm(h, (h.shape[-1],), w["final_norm.weight"], w["final_norm.bias"], 1e-5)


@pytest.mark.parametrize("opts", [OPTS, dict(window=5), dict(sinks=3), dict(rotary_dim=24, rotary_base=500.0),
                                  dict(qk_norm=True)], ids=str)
def test_training_through_the_model(opts):
    """Hidden states and the gradient of every parameter and of the input, float32 against float64."""
    announce("gqa_options", opts=opts)
    m = _model(torch.float32, **opts)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 23, 48, generator=g, dtype=torch.float32)
    do = torch.randn(2, 23, 96, generator=g, dtype=torch.float32)
    xd = x.cuda().requires_grad_()
    out = m.sequence(xd)
    params = dict(m.named_parameters())
    grads = torch.autograd.grad(out, [xd, *params.values()], do.cuda())
    w = {n: p.detach().cpu().double().requires_grad_() for n, p in params.items()}
    xr = x.double().requires_grad_()
    ref = _reference(w, xr, 4, 2, opts)
    want = torch.autograd.grad(ref, [xr, *w.values()], do.double())
    assert_close(host(out), ref.detach().numpy(), 1e-4, "hidden states")
    for name, a, b in zip(["x", *w], grads, want):
        if name.endswith("k_proj.bias") and not opts.get("rotary_dim") and not opts.get("qk_norm"):
            # a key bias shifts a whole softmax row: its gradient is zero, and what the kernel leaves is rounding
            assert float(a.abs().max()) <= 1e-4 * float(b.abs().max() + grads[0].abs().max())
        else:
            assert_close(host(a), b.numpy(), 1e-4, name, elementwise=False)


@pytest.mark.parametrize("opts", [OPTS, {}], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_prompts_and_steps_match_the_whole_sequence(dtype, opts):
    """Ragged prompts padded behind, then single tokens with places that pause, against ``sequence`` on each text."""
    announce("gqa_steps", dtype=dtype, opts=opts)
    m = _model(dtype, **opts)
    g = torch.Generator().manual_seed(2)
    texts = [torch.randn(n, 48, generator=g).to(dtype).cuda() for n in (31, 18, 24)]
    prompt = [13, 1, 7]
    cache = m.paged_cache(3, 40, block_size=4)
    x = torch.zeros(3, 13, 48, dtype=dtype, device="cuda")
    for r, (t, n) in enumerate(zip(texts, prompt)):
        x[r, :n] = t[:n]
    counts = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    h = m.step(x, cache, counts)
    got = [[h[r, i] for i in range(n)] for r, n in enumerate(prompt)]
    at = list(prompt)
    for turn in range(40):
        go = [at[r] < len(t) and (turn + r) % 4 != 0 for r, t in enumerate(texts)]
        x1 = torch.stack([t[min(a, len(t) - 1)] for t, a in zip(texts, at)])[:, None]
        h = m.step(x1, cache, torch.tensor(go, dtype=torch.int32, device="cuda"))
        for r in range(3):
            if go[r]:
                got[r].append(h[r, 0])
                at[r] += 1
    assert not cache.exhausted() and cache.lengths.tolist() == [len(t) for t in texts]
    with torch.no_grad():
        for r, t in enumerate(texts):
            want = m.sequence(t[None])[0]
            # two layers of bf16 products and norms, each side with its own roundings
            assert_close(host(torch.stack(got[r])), host(want), 1e-4 if dtype == torch.float32 else 3e-2, f"text {r}",
                         elementwise=False)


def test_what_the_padding_holds_does_not_matter():
    """Padding of NaN behind ragged prompts, and in a place that takes no tokens: the real tokens' states are finite
    and those of zero padding."""
    announce("gqa_padding")
    m = _model(torch.float32, **OPTS)
    x = torch.randn(3, 9, 48, generator=torch.Generator().manual_seed(4)).cuda()
    counts = torch.tensor([4, 9, 0], dtype=torch.int32, device="cuda")
    pad = (torch.arange(9, device="cuda") >= counts[:, None])[..., None]
    a, b = (m.paged_cache(3, 16, block_size=4) for _ in range(2))
    want = m.step(x.masked_fill(pad, 0.0), a, counts)
    got = m.step(x.masked_fill(pad, math.nan), b, counts)
    assert torch.isfinite(got[~pad[..., 0]]).all() and torch.equal(got[~pad[..., 0]], want[~pad[..., 0]])
    assert torch.equal(a.k[1], b.k[1]) and torch.equal(a.v[0], b.v[0])
    x1 = torch.full((3, 1, 48), math.nan, device="cuda")
    x1[:2] = x[:2, :1]
    one = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
    assert torch.isfinite(m.step(x1, b, one)[:2]).all()


def test_release_and_exhaustion():
    """Pages return to the list and are used again; a list that ends is reported, and its tokens are not stored."""
    announce("paged_cache_release")
    from edifice_amd import blocks
    c = blocks.PagedCache(1, 2, 8, 1, 32, block_size=4, num_blocks=3, dtype=torch.float32)
    counts = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")  # noqa: E731
    c.extend(8, counts(8, 3))
    assert not c.exhausted() and c.table.tolist() == [[0, 1], [2, -1]]
    c.release(0)
    slots, _ = c.extend(5, counts(0, 4))
    assert c.table.tolist() == [[-1, -1], [2, 0]] and not c.exhausted()
    assert slots.tolist()[1] == [11, 0, 1, 2, -1]
    slots, positions = c.extend(8, counts(8, 0))
    assert c.exhausted() and c.table.tolist()[0] == [1, -1]
    assert slots.tolist()[0] == [4, 5, 6, 7, -1, -1, -1, -1] and positions.tolist()[0] == list(range(8))


def test_prompt_into_a_filled_place_is_refused():
    announce("prompt_refused")
    m = _model(torch.float32, **OPTS)
    cache = m.paged_cache(2, 16)
    x = torch.zeros(2, 3, 48, device="cuda")
    m.step(x, cache, torch.tensor([3, 0], device="cuda"))
    with pytest.raises(ValueError):
        m.step(x, cache, torch.tensor([2, 2], device="cuda"))
    m.step(x, cache, torch.tensor([0, 2], device="cuda"))
    assert cache.lengths.tolist() == [3, 2]
    with pytest.raises(ValueError):
        cache.extend(1, torch.tensor([1], device="cuda"))
    with pytest.raises(ValueError):  # texts and places do not match; nothing has moved
        m.step(x[:1, :1], cache)
    assert cache.lengths.tolist() == [3, 2]


def test_captured_step_replays():
    """One decode step captured (cache bookkeeping among it) and replayed against eager steps of a second cache."""
    announce("gqa_captured_step")
    m = _model(torch.bfloat16, **OPTS)
    g = torch.Generator().manual_seed(8)
    a, b = (m.paged_cache(2, 24, block_size=4) for _ in range(2))
    x = torch.randn(2, 1, 48, generator=g).to(torch.bfloat16).cuda()
    for c in (a, b):
        m.step(x, c)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        h = m.step(x, a)
    for _ in range(15):
        x.copy_(torch.randn(2, 1, 48, generator=g).to(torch.bfloat16))
        want = m.step(x, b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, want) and torch.equal(a.table, b.table) and torch.equal(a.lengths, b.lengths)


def test_default_attention_is_unchanged():
    """Without the options the block runs what it ran: flash attention on repeated heads."""
    from edifice_amd import fused_scan as fs
    announce("gqa_default")
    m = _model(torch.bfloat16)
    a = m.blocks[0].attn
    x = torch.randn(2, 9, 96, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()
    sp = lambda t: t.view(2, 9, -1, 24).transpose(1, 2)  # noqa: E731
    q, k, v = sp(a.q_proj(x)), sp(a.k_proj(x)).repeat_interleave(2, 1), sp(a.v_proj(x)).repeat_interleave(2, 1)
    want = a.out_proj(fs.merge_heads(fs.flash_attention(q, k, v, causal=True)))
    assert torch.equal(a(x), want)
