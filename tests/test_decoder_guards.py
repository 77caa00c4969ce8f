"""What the decoder's attention operators and the paged cache do with calls that they refuse or cannot serve, without a
GPU: a refusal leaves the process and the cache as they were."""
import itertools

import pytest
import torch

from edifice_amd import fused_scan as fs
from edifice_amd._native import EdificeHipError, lib

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
