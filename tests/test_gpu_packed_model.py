"""Packed texts and the 8-bit cache run together, as a model uses them: training on texts laid end to end, and prompts,
steps and prompts that go on over both kinds of cache."""
import itertools
import math

import pytest
import torch

from tests.conftest import assert_close
from tests.gpu_util import announce, host
from tests.test_gpu_decoder import OPTS, _model

pytestmark = pytest.mark.gpu
f32, bf16 = torch.float32, torch.bfloat16


def _dev(lengths):
    return torch.tensor(list(itertools.accumulate(lengths, initial=0)), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("opts", [OPTS, {}, dict(rotary_dim=24)], ids=str)
def test_training_on_packed_texts(opts):
    """Hidden states are those of each text alone, and gradients the sums of theirs."""
    announce("packed model", opts=opts)
    m = _model(f32, **opts)
    g = torch.Generator().manual_seed(1)
    lengths = [23, 1, 0, 140, 9]
    x = torch.randn(sum(lengths) + 4, 48, generator=g).cuda().requires_grad_()
    do = torch.randn(sum(lengths), 96, generator=g).cuda()
    params = dict(m.named_parameters())
    got = m.packed(x, _dev(lengths))
    grads = torch.autograd.grad(got[:sum(lengths)], [x, *params.values()], do, retain_graph=False)
    offsets = _dev(lengths).tolist()
    want = torch.cat([m.sequence(x[None, a:b])[0] for a, b in zip(offsets, offsets[1:]) if b > a])
    ref = torch.autograd.grad(want, [x, *params.values()], do)
    assert_close(host(got[:sum(lengths)]), host(want), 1e-4, "hidden states")
    for name, a, b in zip(["x", *params], grads, ref):
        if name.endswith("k_proj.bias") and not opts:
            # a key bias shifts a whole softmax row: its gradient is zero, and what the kernels leave is rounding
            assert float(a.abs().max()) <= 1e-4 * float(grads[0].abs().max())
        else:
            assert_close(host(a), host(b), 1e-4, name, elementwise=False)


def _walk(m, cache, texts, plan):
    """The texts through the cache by ``plan``'s turns (method, tokens of each place); the hidden states of each."""
    at, got = [0] * len(texts), [[] for _ in texts]
    for method, n in plan:
        T = max(1, *n)
        x = torch.full((len(texts), T, texts[0].shape[1]), math.nan if method == "go_on" else 0.0, dtype=texts[0].dtype,
                       device="cuda")
        for r, c in enumerate(n):
            x[r, :c] = texts[r][at[r]:at[r] + c]
        h = getattr(m, method)(x, cache, torch.tensor(n, dtype=torch.int32, device="cuda"))
        for r, c in enumerate(n):
            got[r].append(h[r, :c])
            at[r] += c
            if method == "go_on":
                assert not h[r, c:].any()
    return [torch.cat(g) for g in got], at


PLAN = [("step", (13, 1, 0)), ("go_on", (5, 9, 30)), ("step", (1, 1, 1)), ("step", (0, 1, 1)), ("go_on", (1, 0, 2)),
        ("go_on", (0, 0, 0)), ("go_on", (11, 150, 1)), ("step", (1, 1, 1))]


@pytest.mark.parametrize("opts", [OPTS, {}], ids=str)
@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
def test_prompts_that_go_on_match_the_whole_sequence(dtype, opts):
    announce("go_on", dtype=dtype, opts=opts)
    m = _model(dtype, **opts)
    g = torch.Generator().manual_seed(2)
    texts = [torch.randn(sum(n[r] for _, n in PLAN), 48, generator=g).to(dtype).cuda() for r in range(3)]
    cache = m.paged_cache(3, 200, block_size=4)
    got, at = _walk(m, cache, texts, PLAN)
    assert not cache.exhausted() and cache.lengths.tolist() == at == [len(t) for t in texts]
    with torch.no_grad():
        for r, t in enumerate(texts):
            # two layers of bf16 products and norms, each side with its own roundings
            assert_close(host(got[r]), host(m.sequence(t[None])[0]), 1e-4 if dtype == f32 else 3e-2, f"text {r}",
                         elementwise=False)


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("opts", [OPTS, {}], ids=str)
def test_eight_bit_cache(code, opts):
    """One attention layer with and without an 8-bit cache, its output projection the identity: outputs differ by no more
    than the rounding of keys and values allows.  A key off by dk shifts a score by |q| |dk| / sqrt(d) at most, so each
    probability by a factor within e^(2 shift); a value by dv; o by (e^(2 shift) - 1) max |v| + dv."""
    announce("8-bit cache", code=code, opts=opts)
    from edifice_amd import blocks
    m = _model(f32, **opts)
    attn = m.blocks[0].attn
    with torch.no_grad():
        attn.out_proj.weight.copy_(torch.eye(96))
        attn.out_proj.bias.zero_()
    caches = [blocks.PagedCache(1, 2, 64, 2, 24, block_size=8, dtype=dt) for dt in (f32, code)]
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for n in (20, 1, 1, 13, 1):  # a prompt, tokens, tokens that go on
            x = torch.randn(2, n, 96, generator=g).cuda()
            outs = []
            for c in caches:
                first = not bool(c.lengths.any())
                slots, positions = c.extend(n)
                if first or n == 1:
                    outs.append(attn.step(x, c, 0, slots, positions))
                else:
                    off, keys = _dev([n, n]), _dev(c.lengths.tolist())
                    packed = [t.reshape(1, -1, *t.shape[2:]) for t in (x, slots, positions)]
                    outs.append(attn.go_on(packed[0], c, 0, packed[1], packed[2], off, keys, int(keys[-1])).view(2, n, 96))
            q = attn._heads(x, positions)[0]
            total = _dev(caches[0].lengths.tolist())
            (k, v), (k8, v8) = (c.read(0, total, int(total[-1]), f32) for c in caches)
            dk, dv = (k8 - k).norm(dim=-1).max(), (v8 - v).abs().max()
            shift = q.norm(dim=-1).max() * dk / math.sqrt(24)
            bound = float((torch.exp(2 * shift) - 1) * v.abs().max() + dv) + 1e-5
            assert float((outs[1] - outs[0]).abs().max()) <= bound
            # and the 8-bit cache holds what the other does, to a step of its pages' scales
            limit = v.abs().max() / 127 if code == torch.int8 else v.abs().max() / 16 + v.abs().max() / 448 * 2.0 ** -9
            assert float(dv) <= 2 * float(limit)
    # the whole model on such a cache
    texts = [torch.randn(sum(n[r] for _, n in PLAN), 48, generator=g).cuda() for r in range(3)]
    cache = m.paged_cache(3, 200, block_size=16, dtype=code)
    got, at = _walk(m, cache, texts, PLAN)
    assert cache.lengths.tolist() == at and all(bool(torch.isfinite(t).all()) for t in got)


def test_captured_step_on_an_eight_bit_cache():
    """A decode step captured and replayed against eager steps of a second cache; a released place starts anew."""
    announce("8-bit step captured")
    m = _model(bf16, **OPTS)
    g = torch.Generator().manual_seed(8)
    a, b = (m.paged_cache(2, 24, block_size=4, dtype=torch.int8) for _ in range(2))
    x = torch.randn(2, 1, 48, generator=g).to(bf16).cuda()
    for c in (a, b):
        m.step(x, c)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        h = m.step(x, a)
    for i in range(15):
        if i == 9:
            for c in (a, b):
                c.release(1)
        x.copy_(torch.randn(2, 1, 48, generator=g).to(bf16) * 2.0 ** (i % 5))
        want = m.step(x, b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, want) and torch.equal(a.table, b.table) and torch.equal(a.lengths, b.lengths)
        assert all(torch.equal(p, q) for p, q in zip(a.k_scale + a.k, b.k_scale + b.k))


@pytest.mark.parametrize("kind", [None, torch.int8], ids=str)
def test_no_places(kind):
    """A cache of no places takes steps and prompts that go on, and answers with no states."""
    announce("no places", kind=kind)
    m = _model(f32, **OPTS)
    cache = m.paged_cache(0, 24, block_size=4, **({} if kind is None else dict(dtype=kind)))
    with torch.no_grad():
        width = m.sequence(torch.zeros(1, 1, 48, device="cuda")).shape[2]
    for method, n in (("go_on", 5), ("go_on", 1), ("step", 3), ("step", 1)):
        assert getattr(m, method)(torch.zeros(0, n, 48, device="cuda"), cache).shape == (0, n, width)
