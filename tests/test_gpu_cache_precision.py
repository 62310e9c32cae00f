"""Attention over 4-bit and scored caches, row by row at a tolerance that counts roundings as they add up (cache_norms):
a tile of V left out, taken from elsewhere or read at the wrong place, or P held in fewer bits, exceeds it."""
import pytest
import torch

import fused_attn
from cache_helpers import garbage_behind, gen, oracle
from cache_norms import check_rows, deviation
from helpers import announce

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _floats(shape, seed):
    g = gen(seed)
    return torch.randn(shape, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=g))


def _int4(b, hkv, n, d):
    """(k codes, k pairs, v codes, v pairs) and (k values, v values, what P's rounding meets)."""
    (k4, ks), (v4, vs) = (tuple(t.cuda() for t in fused_attn.quantize_kv_int4(_floats((b, hkv, n, d), i).cpu())) for i in (1, 2))
    return (k4, ks, v4, vs), (oracle.values(k4, ks), oracle.values(v4, vs), deviation(v4, vs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nk", [40, 1000, 1001])
@pytest.mark.parametrize("nq", [1, 4, 8, 16])  # 4, 16, 32 and 64 rows: each number of row blocks
@pytest.mark.parametrize("split", [None, 64, 1024])
def test_int4(dtype, d, nk, nq, split):
    announce(f"int4 norms {dtype} d={d} nk={nk} nq={nq} split={split}")
    q = torch.randn(2, 8, nq, d, device="cuda", generator=gen(nk)).to(dtype)
    args, want = _int4(2, 2, nk, d)
    check_rows(fused_attn.attention_int4(q, *args, causal=True, split_len=split), q, *want, causal=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 6, 16, 40])  # up to 160 rows
@pytest.mark.parametrize("page,split", [(16, None), (48, 64), (256, 1024)])  # of 64: 28 partitions
def test_int4_paged(dtype, d, nq, page, split):
    announce(f"int4 paged norms {dtype} d={d} nq={nq} page={page} split={split}")
    lens = [1750, 1, 97, 0, 1000]
    q = torch.randn(5, 8, nq, d, device="cuda", generator=gen(1)).to(dtype)
    (k4, ks, v4, vs), _ = _int4(5, 2, 1750, d)
    garbage_behind(k4, ks, lens), garbage_behind(v4, vs, lens)
    kp, vp, ksp, vsp, bt, sl = fused_attn.paged_from_dense_int4(k4, ks, v4, vs, page, lens, extra_pages=2,
                                                                generator=torch.Generator().manual_seed(1))
    got = fused_attn.attention_paged(q, kp, vp, bt, sl, causal=True, split_len=split, k_scale=ksp, v_scale=vsp)
    check_rows(got, q, oracle.values(k4, ks), oracle.values(v4, vs), deviation(v4, vs), causal=True, lens=lens)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 6, 30])  # 4, 24 and 120 rows
@pytest.mark.parametrize("split", [64, 128, 1024])  # 40, 20 and 3 partitions: the merges of many and of few
def test_int4_many_partitions_bf16(d, nq, split):
    announce(f"int4 partitions bf16 d={d} nq={nq} split={split}")
    lens = [2500, 1300, 0]
    q = torch.randn(3, 8, nq, d, device="cuda", generator=gen(1)).bfloat16()
    args, want = _int4(3, 2, 2500, d)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for s, n in ((None, None), (sl, lens)):
        got = fused_attn.attention_int4(q, *args, causal=True, seqlens_k=s, split_len=split)
        check_rows(got, q, *want, causal=True, lens=n)


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 4, 8, 40])
@pytest.mark.parametrize("split", [None, 64])
def test_scored(int4, dtype, d, nq, split):
    announce(f"scored norms int4={int4} {dtype} d={d} nq={nq} split={split}")
    lens = [1300, 33, 1000]
    q = torch.randn(3, 8, nq, d, device="cuda", generator=gen(1)).to(dtype)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if int4:
        (k, ks, v, vs), want = _int4(3, 2, 1300, d)
        extra = dict(k_scale=ks, v_scale=vs)
    else:
        k, v, extra = _floats((3, 2, 1300, d), 1).to(dtype), _floats((3, 2, 1300, d), 2).to(dtype), {}
        want = k.double(), v.double()
    got, w = fused_attn.attention_scored(q, k, v, causal=True, seqlens_k=sl, split_len=split, **extra)
    check_rows(got, q, *want, causal=True, lens=lens)
    true = oracle.attention(q, *want[:2], True, lens=lens)[2]
    # a weight's relative error: its scores' (cache_norms: 2^-13.3 at most, as far as it is not shared), and the sum's
    assert ((w.double() - true).norm(dim=-1) <= 2.0 ** -13 * true.norm(dim=-1) + 1e-30).all()
