"""The decoder's attention under the modes that a program switches between: inference and training, eager and captured."""
import pytest
import torch

from edifice_amd import blocks
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

OPTS = dict(rotary_dim=16, qk_norm=True, window=9, sinks=2)


def _model(dtype=torch.float32):
    torch.manual_seed(3)
    return blocks.build("gqa", embed_size=48, hidden_size=96, num_heads=4, num_kv_heads=2, **OPTS).to(device="cuda",
                                                                                                      dtype=dtype)


def test_training_after_inference_mode():
    """A first call under inference_mode, then a backward: the gradients of a model that only trained."""
    announce("gqa_inference_then_training")
    x = torch.randn(2, 11, 48, generator=torch.Generator().manual_seed(0)).cuda()

    def grads(m):
        return torch.autograd.grad(m.sequence(x).square().sum(), list(m.parameters()))
    m = _model()
    with torch.inference_mode():
        m.sequence(x)
        m.step(x, m.paged_cache(2, 16))
    for a, b in zip(grads(m), grads(_model())):
        assert torch.equal(a, b)


def test_first_step_of_a_model_captured():
    """A model's very first step inside a capture (its angles are on the GPU already), replayed against eager steps."""
    announce("gqa_first_step_captured")
    warm = _model(torch.bfloat16)
    warm.step(torch.zeros(2, 1, 48, dtype=torch.bfloat16, device="cuda"), warm.paged_cache(2, 24, block_size=4))
    m = _model(torch.bfloat16)
    a, b = (m.paged_cache(2, 24, block_size=4) for _ in range(2))
    x = torch.zeros(2, 1, 48, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        h = m.step(x, a)
    g = torch.Generator().manual_seed(8)
    for _ in range(6):
        x.copy_(torch.randn(2, 1, 48, generator=g).to(torch.bfloat16))
        want = m.step(x, b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, want) and torch.equal(a.lengths, b.lengths)
