"""What the host code of the 4-bit cache, of scored attention and of eviction accepts and refuses, on the CPU: the library's
own argument checks run, no kernel is launched."""
import contextlib

import pytest
import torch

from fused_attn import _hip


@pytest.fixture
def host_only(monkeypatch):
    """The path of GPU tensors up to the library, with CPU tensors: calls that have nothing to launch, or are refused."""
    monkeypatch.setattr(_hip, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(_hip, "_on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_hip, "_stream", lambda t: 0)


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("b,nq,nk", [(0, 1, 9), (0, 1, 0), (2, 0, 9), (2, 0, 0)])
def test_scored_calls_without_queries(host_only, int4, b, nq, nk):
    q = torch.zeros(b, 4, nq, 64).half()
    k = torch.zeros(b, 2, nk, 32, dtype=torch.uint8) if int4 else torch.zeros(b, 2, nk, 64).half()
    pairs = torch.zeros(b, 2, nk, 2).half() if int4 else None
    o, w = _hip.cache_attention(q, k, k, pairs, pairs, True, 0.1, None, return_scores=True)
    assert o.shape == q.shape and w.shape == (b, 2, nk) and not w.any()
    with pytest.raises(RuntimeError, match="split_len"):
        _hip.cache_attention(q, k, k, pairs, pairs, True, 0.1, 65, return_scores=True)


@pytest.mark.parametrize("cols,nk", [(0, 1), (0, 640), (3, 49)])
def test_paged_calls_need_their_pages(host_only, cols, nk):
    """A table without columns has no address: the call must not become one over a dense cache."""
    q, pool, pairs = torch.zeros(2, 4, 1, 64).half(), torch.zeros(5, 2, 16, 32, dtype=torch.uint8), torch.zeros(5, 2, 16, 2).half()
    table, lens = torch.zeros(2, cols, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="fewer pages"):
        _hip.cache_attention(q, pool, pool, pairs, pairs, True, 0.1, None, seqlens_k=lens, block_table=table, max_seqlen_k=nk)
