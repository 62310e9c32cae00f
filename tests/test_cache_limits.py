"""What the host code of the 4-bit cache, of scored attention and of eviction accepts and refuses, on the CPU: the library's
own argument checks run, no kernel is launched."""
import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import fused_attn
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


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


def _params(**over):
    p = _hip.CacheParams()
    p.q = p.k = p.v = p.o = p.k_scale = p.v_scale = 0x10000  # never dereferenced
    p.batch, p.heads_q, p.heads_kv, p.seqlen_q, p.seqlen_k, p.head_dim = 1, 4, 2, 1, 64, 64
    p.q_stride_b, p.q_stride_h, p.q_stride_n = 256, 64, 64
    p.o_stride_b, p.o_stride_h, p.o_stride_n = 256, 64, 64
    p.k_stride_b, p.k_stride_h, p.k_stride_n = 4096, 2048, 32
    p.v_stride_b, p.v_stride_h, p.v_stride_n = 4096, 2048, 32
    p.scale, p.dtype, p.kv_dtype = 0.125, _hip.BF16, _hip.INT4
    for k, v in over.items():
        setattr(p, k, v)
    return p


PAGED = dict(block_table=0x20000, seqlens_k=0x20000, block_table_cols=1024, block_table_stride=1024, page_size=16, num_pages=4,
             seqlen_k=16384)


@pytest.mark.parametrize("over,split,msg", [
    (PAGED, 4160, "258 pages"),
    (dict(batch=1 << 16, seqlen_q=1 << 13), 64, "grid too large"),  # 2^31 rows
    (dict(batch=1 << 10, seqlen_k=1 << 26), 64, "grid too large"),  # 2^31 partitions
    (dict(scores_out=0x10000, seqlen_q=(1 << 22) + 1), 64, "at most 2^23"),  # their scores' offsets pass 32 bits
])
def test_workspace_query_refuses_what_the_call_refuses(lib, over, split, msg):
    p = _params(**over)
    assert lib.fa_attention_cache_workspace_bytes(p, split) == 0 and msg in lib.fa_last_error().decode()
    assert lib.fa_attention_cache(p, split, 0x10000, 1 << 62, None) == _hip.FA_ERR_UNSUPPORTED
    assert msg in lib.fa_last_error().decode()


def test_workspace_query_at_the_longest_partition(lib):
    assert lib.fa_attention_cache_workspace_bytes(_params(**PAGED), 4096) == 4 * 4 * (64 * 4 + 8)


def test_most_rows_that_are_scored(lib):
    need = lib.fa_attention_cache_workspace_bytes(_params(scores_out=0x10000, seqlen_q=1 << 22), 64)
    rows = 4 << 22  # partials, the rows' LSE, 64 scores a row
    assert need == rows * (64 + 2) * 4 + rows * 4 + rows * 64 * 4


class _Largest(TorchDispatchMode):
    """The most elements of any tensor that an operator gives."""
    numel = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        got = func(*args, **(kwargs or {}))
        for t in got if isinstance(got, (tuple, list)) else (got,):
            if isinstance(t, torch.Tensor):
                self.numel = max(self.numel, t.numel())
        return got


@pytest.mark.parametrize("nq,causal", [(1, False), (3, True)])
def test_torch_forms_grow_with_the_keys_not_their_square(nq, causal):
    n, hq, hkv, d = 2000, 4, 2, 64
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(1, hq, nq, d, generator=gen).half()
    (k4, ks), (v4, vs) = (fused_attn.quantize_kv_int4(torch.randn(1, hkv, n, d, generator=gen)) for _ in "kv")
    for call in (lambda: fused_attn.attention_int4(q, k4, ks, v4, vs, causal=causal),
                 lambda: fused_attn.attention_scored(q, k4, v4, causal=causal, k_scale=ks, v_scale=vs)):
        with _Largest() as largest:
            call()
        assert largest.numel <= hq * n * d  # a kv-head's rows for each of its q-heads


def _bytes_of(t):
    """Every byte address of t."""
    at = torch.zeros(t.shape, dtype=torch.int64) + t.data_ptr()
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at = at + (torch.arange(n) * s * t.element_size()).view(-1, *[1] * (t.dim() - 1 - i))
    return {a + i for a in at.flatten().tolist() for i in range(t.element_size())}


def test_evict_out_in_parts_of_one_buffer():
    """Outputs between each other's or the caches' rows are taken; memory that is shared is not."""
    scores, k, v = torch.rand(2, 3, 9), torch.randn(2, 3, 9, 4).half(), torch.randn(2, 3, 9, 4).half()
    (wk, wv), _, _, _ = fused_attn.evict_kv(scores, (k, v), 5, 1)
    rows, heads, keys = torch.zeros(2, 3, 6, 2, 4).half(), torch.zeros(2, 6, 5, 4).half(), torch.zeros(2, 3, 14, 4).half()
    apart = [(rows[..., 0, :], rows[..., 1, :]), (heads[:, :3], heads[:, 3:]), (keys[:, :, :5], keys[:, :, 9:]),
             (heads[:, ::2], heads[:, 1::2]), (rows[:, :, :5, 1], heads[:, 3:])]
    for out in apart:
        assert not _bytes_of(out[0]) & _bytes_of(out[1])
        got = fused_attn.evict_kv(scores, (k, v), 5, 1, out=out)[0]
        assert torch.equal(got[0][:, :, :5], wk) and torch.equal(got[1][:, :, :5], wv)
    both = torch.zeros(2, 3, 14, 4).half()  # a cache and its output in one buffer
    both[:, :, 5:] = k
    got = fused_attn.evict_kv(scores, (both[:, :, 5:],), 5, 1, out=(both[:, :, :5],))[0][0]
    assert torch.equal(got, wk) and torch.equal(both[:, :, 5:], k)
    shared = [(rows[..., 0, :], rows[..., 0, :]), (heads[:, :3], heads[:, 2:5]), (keys[:, :, :5], keys[:, :, 4:9]),
              (rows.view(2, 3, 6, 8)[..., :4], rows.view(2, 3, 6, 8)[..., 2:6])]
    for out in shared:
        assert _bytes_of(out[0]) & _bytes_of(out[1])
        with pytest.raises(RuntimeError, match="share memory"):
            fused_attn.evict_kv(scores, (k, v), 5, 1, out=out)


def test_apart_never_misses_a_shared_byte():
    gen = torch.Generator().manual_seed(3)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=gen))  # noqa: E731
    buffer, seen = torch.zeros(4000, dtype=torch.uint8), 0
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [pick(1, 4) for _ in range(4)]
            stride = [pick(0, 5) * pick(1, 40) for _ in range(3)] + [1]
            views.append(buffer.as_strided(shape, stride, pick(0, 200)))
        if _hip._apart(*views):
            seen += 1
            assert not _bytes_of(views[0]) & _bytes_of(views[1])
    assert seen > 300


@pytest.mark.parametrize("stride", [(60, 20, 3, 1), (60, 16, 4, 1), (40, 20, 4, 1), (4, 6, 40, 1)])
def test_evict_refuses_an_output_whose_rows_overlap(stride):
    out = torch.zeros(400).as_strided((2, 3, 5, 4), stride)
    with pytest.raises(RuntimeError, match="overlap"):
        fused_attn.evict_kv(torch.rand(2, 3, 9), (torch.randn(2, 3, 9, 4),), 5, 1, out=(out,))


@pytest.mark.parametrize("stride", [(60, 20, 4, 1), (12, 4, 24, 1), (4, 8, 24, 1), (4, 8, 40, 1), (100, 33, 6, 1)])
def test_evict_takes_outputs_of_any_order(stride):
    scores, k = torch.rand(2, 3, 9), torch.randn(2, 3, 9, 4)
    out = torch.zeros(400).as_strided((2, 3, 5, 4), stride)
    assert torch.equal(fused_attn.evict_kv(scores, (k,), 5, 1, out=(out,))[0][0], fused_attn.evict_kv(scores, (k,), 5, 1)[0][0])
