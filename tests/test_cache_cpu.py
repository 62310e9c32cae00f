"""The 4-bit cache, scored attention and eviction on CPU tensors (their torch forms), what they refuse, and the C ABI's
refusals.  Nothing here reaches a kernel launch."""
import ctypes
import math

import numpy as np
import pytest
import torch

import fused_attn
from fused_attn import _hip
from oracle import cache_oracle as cor


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _cache(b, hkv, n, d, seed=0):
    return fused_attn.quantize_kv_int4(torch.randn(b, hkv, n, d, generator=_gen(seed)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [2, 64, 128])
def test_quantize_and_dequantize_match_the_oracle(dtype, d):
    x = (torch.randn(2, 3, 11, d, generator=_gen()) * 3 + 1).to(dtype)
    codes, pairs = fused_attn.quantize_kv_int4(x)
    code, scale, zero = cor.encode(x)
    assert codes.dtype == torch.uint8 and pairs.dtype == torch.float16
    assert np.array_equal(codes.numpy(), cor.pack(code))
    assert np.array_equal(pairs.numpy(), np.stack([scale, zero], -1))
    want = cor.values(codes, pairs)
    assert torch.equal(fused_attn.dequantize_kv_int4(codes, pairs), want.float())
    assert torch.equal(fused_attn.dequantize_kv_int4(codes, pairs, torch.float16), want.float().half())


def test_rows_with_infinities_nan_and_nothing_to_tell_apart():
    x = torch.randn(1, 1, 5, 64, generator=_gen())
    x[0, 0, 0, 3] = math.inf
    x[0, 0, 1, 4] = -math.inf
    x[0, 0, 2, 5] = math.nan
    x[0, 0, 3] = -2.0
    codes, pairs = fused_attn.quantize_kv_int4(x)
    y = fused_attn.dequantize_kv_int4(codes, pairs)[0, 0]
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[1]).all() and y[0].max() > 6e4 and y[1].min() < -6e4
    assert torch.isnan(y[2]).all() and torch.equal(y[3], x[0, 0, 3])
    code, scale, zero = cor.encode(x)
    assert np.array_equal(codes.numpy(), cor.pack(code))


def test_quantize_out_writes_a_slice_only():
    cache = torch.full((2, 2, 10, 32), 7, dtype=torch.uint8), torch.full((2, 2, 10, 2), 7.0, dtype=torch.float16)
    x = torch.randn(2, 2, 3, 64, generator=_gen())
    got = fused_attn.quantize_kv_int4(x, out=tuple(t[:, :, 4:7] for t in cache))
    want = fused_attn.quantize_kv_int4(x)
    for c, g, w in zip(cache, got, want):
        assert torch.equal(c[:, :, 4:7], w) and torch.equal(g, w)
        assert (c[:, :, :4] == 7).all() and (c[:, :, 7:] == 7).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [None, [9, 0], [3, 100], [-1, 1]])
def test_attention_and_scores_match_the_oracle(lens, causal):
    q = torch.randn(2, 4, 3, 64, generator=_gen(1)).half()
    (k4, ks), (v4, vs) = _cache(2, 2, 9, 64, 2), _cache(2, 2, 9, 64, 3)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    o, lse, w = cor.attention(q, cor.values(k4, ks), cor.values(v4, vs), causal, lens=lens)
    got, got_lse = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=causal, seqlens_k=sl, return_lse=True)
    torch.testing.assert_close(got.double(), o, atol=2e-3, rtol=2e-3)
    torch.testing.assert_close(got_lse.double(), lse, atol=1e-4, rtol=1e-4)
    before = torch.rand(2, 2, 9, generator=_gen(4))
    got, scores = fused_attn.attention_scored(q, k4, v4, scores=before, causal=causal, seqlens_k=sl, k_scale=ks, v_scale=vs)
    torch.testing.assert_close(scores.double(), before.double() + w, atol=1e-5, rtol=1e-5)
    k, v = (fused_attn.dequantize_kv_int4(*c, torch.float16) for c in ((k4, ks), (v4, vs)))
    got, scores = fused_attn.attention_scored(q, k, v, causal=causal, seqlens_k=sl)
    o, _, w = cor.attention(q, k, v, causal, lens=lens)
    torch.testing.assert_close(got.double(), o, atol=2e-3, rtol=2e-3)
    torch.testing.assert_close(scores.double(), w, atol=1e-5, rtol=1e-5)


def test_paged_attention_and_append():
    b, hkv, n, d, page = 3, 2, 40, 64, 16
    (k4, ks), (v4, vs) = _cache(b, hkv, n, d, 1), _cache(b, hkv, n, d, 2)
    q = torch.randn(b, 4, 1, d, generator=_gen(3)).half()
    kp, vp, ksp, vsp, bt, sl = fused_attn.paged_from_dense_int4(k4, ks, v4, vs, page, seqlens=[40, 0, 17], extra_pages=2,
                                                                generator=_gen(4))
    want = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=True, seqlens_k=sl)
    got = fused_attn.attention_paged(q, kp, vp, bt, sl, causal=True, k_scale=ksp, v_scale=vsp)
    assert torch.equal(got, want)
    new = torch.randn(b, hkv, 2, d, generator=_gen(5)), torch.randn(b, hkv, 2, d, generator=_gen(6))
    dense = [t.clone() for t in (k4, ks, v4, vs)]
    fused_attn.append_kv_int4(*new, *dense, sl)
    fused_attn.append_kv_int4(*new, kp, ksp, vp, vsp, sl, block_table=bt)
    for x, codes, pairs, pool in ((new[0], *dense[:2], kp), (new[1], *dense[2:], vp)):
        c, s = fused_attn.quantize_kv_int4(x)
        assert torch.equal(codes[1, :, 0:2], c[1]) and torch.equal(pairs[2, :, 17:19], s[2])
        assert torch.equal(pool[bt[2, 1].item(), :, 1:3], c[2])
    assert torch.equal(dense[0][0], k4[0])  # sequence 0 is full: nothing was written


@pytest.mark.parametrize("lens", [None, [20, 3, 0]])
@pytest.mark.parametrize("keep,recent", [(0, 0), (5, 0), (5, 2), (5, 5), (20, 3), (30, 1)])
def test_evict_matches_the_oracle(lens, keep, recent):
    scores = torch.randint(0, 6, (3, 2, 20), generator=_gen(keep)).float()  # many ties
    scores[0, 0, 3], scores[0, 1, 4] = math.nan, math.inf
    k, v = torch.randn(3, 2, 20, 8, generator=_gen(1)), torch.randint(0, 99, (3, 2, 20, 2, 3), dtype=torch.uint8)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    (k2, v2), s2, index, left = fused_attn.evict_kv(scores, (k, v), keep, recent, sl)
    rows = min(keep, 20)
    assert k2.shape == (3, 2, rows, 8) and v2.shape == (3, 2, rows, 2, 3) and index.dtype == torch.int32
    for b in range(3):
        n = 20 if lens is None else lens[b]
        assert left[b] == min(n, keep)
        for h in range(2):
            at = cor.kept(scores[b, h].numpy(), n, keep, recent)
            assert index[b, h].tolist() == at + [-1] * (rows - len(at))
            assert torch.equal(k2[b, h, :len(at)], k[b, h, at]) and torch.equal(v2[b, h, :len(at)], v[b, h, at])
            assert torch.equal(s2[b, h, :len(at)].nan_to_num(7), scores[b, h, at].nan_to_num(7))
            assert (k2[b, h, len(at):] == 0).all() and (s2[b, h, len(at):] == 0).all()


def test_evict_out_leaves_further_rows():
    scores, k = torch.rand(1, 2, 12, generator=_gen()), torch.randn(1, 2, 12, 4, generator=_gen(1))
    out = torch.full((1, 2, 9, 4), 5.0)
    (got,), _, index, _ = fused_attn.evict_kv(scores, [k], 6, 1, out=[out])
    assert got is out and (out[:, :, 6:] == 5).all()
    assert torch.equal(out[0, 1, :6], k[0, 1, index[0, 1].long()])


# ---- refusals ---------------------------------------------------------------------------------------------------


def _attend_args():
    k4, ks = _cache(2, 2, 8, 64)
    return dict(q=torch.zeros(2, 4, 1, 64, dtype=torch.float16), k4=k4, k_scale=ks, v4=k4.clone(), v_scale=ks.clone())


@pytest.mark.parametrize("change,msg", [
    (dict(q=torch.zeros(2, 4, 1, 64)), "q must be"),
    (dict(q=torch.zeros(2, 4, 1, 128, dtype=torch.float16)), "head_dim"),
    (dict(q=torch.zeros(2, 3, 1, 64, dtype=torch.float16)), "multiple"),
    (dict(q=torch.zeros(3, 4, 1, 64, dtype=torch.float16)), "batch"),
    (dict(k4=torch.zeros(2, 2, 8, 32, dtype=torch.int8)), "dtypes|4-bit|head_dim|same"),
    (dict(v4=torch.zeros(2, 2, 7, 32, dtype=torch.uint8), v_scale=torch.zeros(2, 2, 7, 2, dtype=torch.float16)), "shape"),
    (dict(k_scale=torch.zeros(2, 2, 8, 2)), "float16"),
    (dict(k_scale=torch.zeros(2, 2, 8, dtype=torch.float16)), "float16"),
    (dict(v_scale=None), "scale of v"),
    (dict(seqlens_k=torch.zeros(3, dtype=torch.int32)), "seqlens_k"),
    (dict(seqlens_k=torch.zeros(2, dtype=torch.int64)), "seqlens_k"),
])
def test_attention_int4_refuses(change, msg):
    with pytest.raises(RuntimeError, match=msg):
        fused_attn.attention_int4(**{**_attend_args(), **change})


@pytest.mark.parametrize("change,msg", [
    (dict(scores=torch.zeros(2, 2, 7)), "scores"),
    (dict(scores=torch.zeros(2, 2, 8, dtype=torch.float16)), "scores"),
    (dict(k_scale=torch.zeros(2, 2, 8, 2, dtype=torch.float16)), "belong"),
    (dict(v=torch.zeros(2, 2, 9, 64, dtype=torch.float16)), "same shape"),
    (dict(v=torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)), "dtype"),
    (dict(q=torch.zeros(2, 4, 1, 64)), "q must be"),
])
def test_attention_scored_refuses(change, msg):
    kv = torch.zeros(2, 2, 8, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match=msg):
        fused_attn.attention_scored(**{**dict(q=torch.zeros(2, 4, 1, 64, dtype=torch.float16), k=kv, v=kv), **change})


@pytest.mark.parametrize("x", [torch.zeros(2, 3, 64), torch.zeros(1, 1, 2, 63), torch.zeros(1, 1, 2, 64, dtype=torch.int32)])
def test_quantize_refuses(x):
    with pytest.raises(RuntimeError):
        fused_attn.quantize_kv_int4(x)


def test_quantize_out_refuses_other_shapes():
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="shape"):
        fused_attn.quantize_kv_int4(x, out=(torch.zeros(1, 2, 4, 32, dtype=torch.uint8), torch.zeros(1, 2, 4, 2).half()))
    with pytest.raises(RuntimeError, match="float16"):
        fused_attn.quantize_kv_int4(x, out=(torch.zeros(1, 2, 3, 32, dtype=torch.uint8), torch.zeros(1, 2, 3, 2)))


@pytest.mark.parametrize("change,msg", [
    (dict(v=torch.zeros(2, 2, 2, 64)), "same shape"),
    (dict(k=torch.zeros(2, 2, 1, 128), v=torch.zeros(2, 2, 1, 128)), "fit"),
    (dict(k=torch.zeros(3, 2, 1, 64), v=torch.zeros(3, 2, 1, 64)), "fit"),
    (dict(seqlens_k=torch.zeros(2)), "seqlens_k"),
    (dict(block_table=torch.zeros(3, 1, dtype=torch.int32)), "block_table"),
    (dict(k_scale=torch.zeros(2, 2, 8, 2)), "float16"),
    (dict(k_cache=torch.zeros(2, 2, 8, 64, dtype=torch.uint8)[..., ::2]), "stride"),
    (dict(k_scale=torch.zeros(2, 2, 8, 3, dtype=torch.float16)[..., :2]), "stride"),
    (dict(k_cache=torch.zeros(2, 2, 1, 32, dtype=torch.uint8).expand(2, 2, 8, 32)), "stride"),
])
def test_append_refuses(change, msg):
    k4, ks = _cache(2, 2, 8, 64)
    args = dict(k=torch.zeros(2, 2, 1, 64), v=torch.zeros(2, 2, 1, 64), k_cache=k4, k_scale=ks, v_cache=k4.clone(),
                v_scale=ks.clone(), seqlens_k=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match=msg):
        fused_attn.append_kv_int4(**{**args, **change})


@pytest.mark.parametrize("change,msg", [
    (dict(scores=torch.zeros(2, 8)), "scores"),
    (dict(scores=torch.zeros(2, 2, 8, dtype=torch.float64)), "scores"),
    (dict(caches=[torch.zeros(2, 2, 7, 4)]), "cache must be"),
    (dict(caches=[torch.zeros(2, 2, 8, 0)]), "rows"),
    (dict(caches=[torch.zeros(2, 2, 8, 1)] * 9), "at most 8"),
    (dict(recent=5), "recent"),
    (dict(recent=-1), "recent"),
    (dict(keep=-1), "recent"),
    (dict(seqlens_k=torch.zeros(2, 1, dtype=torch.int32)), "seqlens_k"),
    (dict(out=[]), "out must hold"),
    (dict(out=[torch.zeros(2, 2, 3, 4)]), "at least 4 rows"),
    (dict(out=[torch.zeros(2, 2, 4, 4, dtype=torch.float16)]), "its type"),
    (dict(out=[torch.zeros(2, 2, 1, 4).expand(2, 2, 4, 4)]), "strides"),
    (dict(out=[torch.zeros(2, 2, 4, 8)[..., ::2]]), "contiguous rows"),
])
def test_evict_refuses(change, msg):
    args = dict(scores=torch.zeros(2, 2, 8), caches=[torch.zeros(2, 2, 8, 4)], keep=4, recent=1)
    with pytest.raises(RuntimeError, match=msg):
        fused_attn.evict_kv(**{**args, **change})


def test_evict_refuses_shared_memory():
    k = torch.zeros(2, 2, 8, 4)
    for out in ([k[:, :, :4]], [k]):
        with pytest.raises(RuntimeError, match="share memory"):
            fused_attn.evict_kv(torch.zeros(2, 2, 8), [k], 4, out=out)
    two = torch.zeros(2, 2, 8, 4)
    with pytest.raises(RuntimeError, match="share memory"):
        fused_attn.evict_kv(torch.zeros(2, 2, 8), [k, k], 4, out=[two, two])


# ---- C ABI ---------------------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


def test_struct_sizes():
    assert ctypes.sizeof(_hip.Int4Params) == 120 and ctypes.sizeof(_hip.Int4AppendParams) == 288
    assert ctypes.sizeof(_hip.CacheParams) == 344 and ctypes.sizeof(_hip.EvictTensor) == 72
    assert ctypes.sizeof(_hip.EvictParams) == 80 + 8 * 72


def _cache_params(**over):
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


PAGED = dict(block_table=0x20000, seqlens_k=0x20000, block_table_cols=4, block_table_stride=4, page_size=16, num_pages=4)


@pytest.mark.parametrize("over,code,msg", [
    (dict(head_dim=32), _hip.FA_ERR_UNSUPPORTED, "head_dim"),
    (dict(dtype=_hip.F32), _hip.FA_ERR_UNSUPPORTED, "dtype"),
    (dict(kv_dtype=_hip.F16), _hip.FA_ERR_INVALID_ARGUMENT, "4-bit"),
    (dict(kv_dtype=_hip.BF16), _hip.FA_ERR_UNSUPPORTED, "scores"),
    (dict(kv_dtype=_hip.FP8_E4M3), _hip.FA_ERR_INVALID_ARGUMENT, "4-bit"),
    (dict(heads_q=3), _hip.FA_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(seqlen_k=-1), _hip.FA_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(seqlen_k=(1 << 30) + 1), _hip.FA_ERR_UNSUPPORTED, "2\\^30"),
    (dict(scale=math.nan), _hip.FA_ERR_INVALID_ARGUMENT, "finite"),
    (dict(scale=math.inf), _hip.FA_ERR_INVALID_ARGUMENT, "finite"),
    (dict(scale=-2e30), _hip.FA_ERR_INVALID_ARGUMENT, "1e30"),
    (dict(k_scale_stride_n=1 << 22), _hip.FA_ERR_UNSUPPORTED, "scale token stride"),
    (dict(v_scale_stride_n=-1), _hip.FA_ERR_UNSUPPORTED, "scale token stride"),
    (dict(k=0), _hip.FA_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(k_scale=0), _hip.FA_ERR_INVALID_ARGUMENT, "k_scale"),
    (dict(k=0x10008), _hip.FA_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(v_scale=0x10002), _hip.FA_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(k_stride_n=40), _hip.FA_ERR_INVALID_ARGUMENT, "k/v strides"),
    (dict(q_stride_h=60), _hip.FA_ERR_INVALID_ARGUMENT, "q strides"),
    (dict(o_stride_n=62), _hip.FA_ERR_INVALID_ARGUMENT, "o strides"),
    (dict(v_stride_n=1 << 24), _hip.FA_ERR_UNSUPPORTED, "token stride"),
    (dict(lse=0x20000, lse_stride_h=-1), _hip.FA_ERR_INVALID_ARGUMENT, "LSE"),
    (dict(PAGED, seqlens_k=0), _hip.FA_ERR_INVALID_ARGUMENT, "seqlens_k"),
    (dict(PAGED, page_size=24), _hip.FA_ERR_INVALID_ARGUMENT, "page_size"),
    (dict(PAGED, num_pages=0), _hip.FA_ERR_INVALID_ARGUMENT, "page"),
    (dict(PAGED, block_table_cols=3), _hip.FA_ERR_INVALID_ARGUMENT, "fewer pages"),
    (dict(PAGED, scores_out=0x20000), _hip.FA_ERR_UNSUPPORTED, "dense"),
])
def test_cache_attention_validation(lib, over, code, msg):
    import re

    p = _cache_params(**over)
    assert lib.fa_attention_cache(p, 64, 0x10000, 1 << 30, None) == code
    assert re.search(msg, lib.fa_last_error().decode())
    assert lib.fa_attention_cache_workspace_bytes(p, 64) == 0


def test_cache_attention_split_len_and_workspace(lib):
    for split in (0, 32, 96, -64):
        assert lib.fa_attention_cache(_cache_params(), split, 0x10000, 1 << 30, None) == _hip.FA_ERR_INVALID_ARGUMENT
        assert "split_len" in lib.fa_last_error().decode()
    need = lib.fa_attention_cache_workspace_bytes(_cache_params(), 64)
    assert need == 4 * (64 * 4 + 8)
    scored = _cache_params(scores_out=0x10000, seqlen_k=65)
    # two partitions, the rows' LSE, and 96 scores a row
    assert lib.fa_attention_cache_workspace_bytes(scored, 64) == 2 * 4 * (64 * 4 + 8) + 16 + 4 * 96 * 4
    assert lib.fa_attention_cache(_cache_params(), 64, 0x10000, need - 1, None) == _hip.FA_ERR_WORKSPACE
    assert lib.fa_attention_cache(_cache_params(), 64, None, need, None) == _hip.FA_ERR_WORKSPACE
    assert lib.fa_attention_cache(_cache_params(), 64, 0x10008, need, None) == _hip.FA_ERR_WORKSPACE
    assert lib.fa_attention_cache(_cache_params(batch=0), 64, None, 0, None) == _hip.FA_OK
    assert lib.fa_attention_cache(None, 64, None, 0, None) == _hip.FA_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over,msg", [
    (dict(keep=9), "keep"), (dict(recent=5), "recent"), (dict(num_tensors=9), "num_tensors"), (dict(seqlen=-1), "sizes"),
    (dict(scores=0), "scores"), (dict(index=0), "index"), (dict(seqlens_out=0), "seqlens_out"),
    (dict(scores=0x10002), "aligned"),
])
def test_evict_validation(lib, over, msg):
    p = _hip.EvictParams()
    p.scores = p.index = p.scores_out = p.seqlens_out = 0x10000
    p.batch, p.heads, p.seqlen, p.keep, p.recent = 1, 1, 8, 4, 0
    for k, v in over.items():
        setattr(p, k, v)
    assert lib.fa_evict_kv(p, None, 0, None) == _hip.FA_ERR_INVALID_ARGUMENT
    assert msg in lib.fa_last_error().decode()


def test_evict_workspace(lib):
    p = _hip.EvictParams()
    p.scores = p.index = p.scores_out = p.seqlens_out = 0x10000
    p.batch, p.heads, p.seqlen, p.keep, p.recent = 2, 3, 8192, 4, 0
    assert lib.fa_evict_kv_workspace_bytes(p) == 0
    for n, groups in ((8193, 2), (65536, 8), (16 * 8192, 16), (16 * 8192 + 1, 9), (33 * 8192, 11)):
        p.seqlen = n  # the counts of 2048 digits a workgroup, and a list of every key
        need = lib.fa_evict_kv_workspace_bytes(p)
        assert need == 6 * (groups * 2048 + n) * 4
        for ws, got in ((0x10000, need - 1), (None, need), (0x10008, need)):
            assert lib.fa_evict_kv(p, ws, got, None) == _hip.FA_ERR_WORKSPACE
    assert lib.fa_evict_kv(None, None, 0, None) == _hip.FA_ERR_INVALID_ARGUMENT
    assert lib.fa_evict_kv_workspace_bytes(None) == 0


@pytest.mark.parametrize("over,code,msg", [
    (dict(head_dim=32), _hip.FA_ERR_UNSUPPORTED, "head_dim"),
    (dict(dtype=_hip.FP8_E4M3), _hip.FA_ERR_UNSUPPORTED, "x must"),
    (dict(x=0), _hip.FA_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(x=0x10008), _hip.FA_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(codes=0x10002), _hip.FA_ERR_INVALID_ARGUMENT, "aligned"),
    (dict(codes_stride_n=30), _hip.FA_ERR_INVALID_ARGUMENT, "words"),
    (dict(scale_stride_n=-1), _hip.FA_ERR_INVALID_ARGUMENT, "negative"),
    (dict(seqlen=-1), _hip.FA_ERR_INVALID_ARGUMENT, "non-negative"),
])
def test_int4_row_validation(lib, over, code, msg):
    p = _hip.Int4Params(0x10000, 512, 512, 64, 1, 1, 8, 64, _hip.BF16, 0, 0x10000, 256, 256, 32, 0x10000, 8, 8, 1)
    for k, v in over.items():
        setattr(p, k, v)
    for f in (lib.fa_quantize_kv_int4, lib.fa_dequantize_kv_int4):
        assert f(p, None) == code
        assert msg in lib.fa_last_error().decode()
    a = _hip.Int4AppendParams(p, p, 0x10000, 8)
    assert lib.fa_append_kv_int4(a, None) == code


def test_append_validation(lib):
    p = _hip.Int4Params(0x10000, 512, 512, 64, 1, 1, 1, 64, _hip.BF16, 0, 0x10000, 256, 256, 32, 0x10000, 8, 8, 1)
    q = _hip.Int4Params.from_buffer_copy(p)
    q.head_dim = 128
    for args, msg in (((p, q, 0x10000, 8), "same sizes"), ((p, p, None, 8), "seqlens_k"), ((p, p, 0x10000, -1), "capacity")):
        assert lib.fa_append_kv_int4(_hip.Int4AppendParams(*args), None) == _hip.FA_ERR_INVALID_ARGUMENT
        assert msg in lib.fa_last_error().decode()
    a = _hip.Int4AppendParams(p, p, 0x10000, 0, 0x10000, 1, 1, 0, 4)
    assert lib.fa_append_kv_int4(a, None) == _hip.FA_ERR_INVALID_ARGUMENT and "page_size" in lib.fa_last_error().decode()
