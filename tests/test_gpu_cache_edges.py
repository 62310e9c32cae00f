"""Edges of the 4-bit cache, of scored attention and of eviction on the GPU: infinities and NaN in operands, calls without
work, other head dims, outputs inside larger buffers, repeated calls."""
import math

import numpy as np
import pytest
import torch

import fused_attn
from cache_helpers import cache, gen, oracle, rows
from helpers import announce

pytestmark = pytest.mark.gpu


def _exactly(codes, pairs, x):
    code, scale, zero = oracle.encode(x)
    assert torch.equal(codes.cpu(), torch.from_numpy(oracle.pack(code)))
    assert torch.equal(pairs.cpu(), torch.from_numpy(np.stack([scale, zero], -1)))


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("nq", [1, 5, 20])  # 4, 20 and 80 rows
def test_nan_query_rows_stay_their_own(int4, nq):
    """A NaN in one q row: its output is NaN, the others' are what they are without it; its kv-head's visible keys score NaN."""
    announce(f"nan query int4={int4} nq={nq}")
    d, n = 128, 300
    q = torch.randn(2, 8, nq, d, device="cuda", generator=gen(1)).bfloat16()
    if int4:
        (k, ks), (v, vs) = cache(2, 2, n, d, 1), cache(2, 2, n, d, 2)
        extra = dict(k_scale=ks, v_scale=vs)
    else:
        k, v, extra = rows((2, 2, n, d), torch.bfloat16, 1), rows((2, 2, n, d), torch.bfloat16, 2), {}
    want, w0 = fused_attn.attention_scored(q, k, v, causal=True, split_len=64, **extra)
    bad = q.clone()
    bad[1, 5, 0, 7] = math.nan
    got, w = fused_attn.attention_scored(bad, k, v, causal=True, split_len=64, **extra)
    assert torch.isnan(got[1, 5, 0]).all()
    got[1, 5, 0] = want[1, 5, 0]
    # (the running maximum is renewed where the NaN is, so p is rounded elsewhere: two roundings of bf16)
    assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * (want.float().abs() + want.float().abs().amax())).all()
    seen = n - nq + 1
    assert torch.isnan(w[1, 1, :seen]).all()
    w[1, 1] = w0[1, 1]
    assert ((w - w0).abs() <= 1e-4 * w0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 16])
def test_scored_16_bit_infinite_and_nan_keys(dtype, d, nq):
    """A key whose score is -inf weighs nothing, wherever it lies in a tile; one that is NaN makes the rows that see it NaN;
    behind a sequence's keys nothing is read; an infinite value is infinite in its channel."""
    announce(f"scored infinite keys {dtype} d={d} nq={nq}")
    n = 200
    q = torch.rand(1, 4, nq, d, device="cuda", generator=gen(1)).to(dtype) + 0.5
    k, v = rows((1, 2, n, d), dtype, 1), rows((1, 2, n, d), dtype, 2)
    low = k.clone()
    gone = [0, 31, 32, 130]
    low[:, :, gone, 3] = -math.inf
    keep = [j for j in range(n) if j not in gone]
    o, _, w = oracle.attention(q, k.double()[:, :, keep], v.double()[:, :, keep])
    got, s = fused_attn.attention_scored(q, low, v, split_len=64)
    tol = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10  # output and P: half a step each
    assert ((got.double() - o).abs() <= tol * v.double().abs().amax()).all()
    assert (s[:, :, gone] == 0).all() and ((s[:, :, keep].double() - w).abs() <= 1e-4 * w + 1e-30).all()
    low[:, :, :64, 3] = -math.inf  # a whole partition
    got, s = fused_attn.attention_scored(q, low[:, :, :130], v[:, :, :130], split_len=64)
    o, _, w = oracle.attention(q, k.double()[:, :, 64:130], v.double()[:, :, 64:130])
    assert ((got.double() - o).abs() <= tol * v.double().abs().amax()).all() and (s[:, :, :64] == 0).all()
    bad = k.clone()
    bad[:, :, n - 1, 5] = math.nan
    got, s = fused_attn.attention_scored(q, bad, v, causal=True, split_len=64)
    assert torch.isnan(got[:, :, -1]).all() and torch.isfinite(got[:, :, :-1]).all() and torch.isnan(s).all()
    sl = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    got, s = fused_attn.attention_scored(q, bad, v, causal=True, seqlens_k=sl, split_len=64)
    assert torch.isfinite(got).all() and torch.isfinite(s).all()
    far = v.clone()
    far[:, :, 70, 9] = math.inf
    got, s = fused_attn.attention_scored(q, k * 0.01, far, split_len=64)
    assert torch.isinf(got[..., 9]).all() and torch.isfinite(s).all()
    got[..., 9] = 0
    assert torch.isfinite(got).all()


def test_calls_repeat_bit_for_bit():
    """Every kernel of a call adds in one order: calls on other inputs in between change nothing."""
    announce("cache repeat")
    for int4 in (False, True):
        for hq, nq, d, lens in ((32, 1, 128, None), (32, 16, 256, None), (64, 1, 64, [3000, 77, 1500]), (8, 32, 128, None)):
            (k4, ks), (v4, vs) = cache(3, 8, 3000, d, 1), cache(3, 8, 3000, d, 2)
            k, v, extra = (k4, v4, dict(k_scale=ks, v_scale=vs)) if int4 else \
                (rows((3, 8, 3000, d), torch.bfloat16, 1), rows((3, 8, 3000, d), torch.bfloat16, 2), {})
            q = [torch.randn(3, hq, nq, d, device="cuda", generator=gen(i)).bfloat16() for i in range(2)]
            sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
            call = lambda x: fused_attn.attention_scored(x, k, v, causal=True, seqlens_k=sl, **extra)  # noqa: E731
            first = call(q[0])
            for _ in range(3):
                call(q[1])
                again = call(q[0])
                assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_writer_with_one_channel_far_beyond_the_others(dtype, d):
    """Finite values whose quotient by the row's scale leaves fp32: their code is 15 (or 0), as for any value past the ends."""
    announce(f"int4 far values {dtype} d={d}")
    x = torch.randn(1, 1, 12, d, device="cuda", generator=gen(1)) * 0.001
    x[0, 0, 0] = 65503.0
    x[0, 0, 0, 5] = 3e38
    x[0, 0, 1] = 65504.0  # (no room above: the scale is 0)
    x[0, 0, 1, 5] = 3e38
    x[0, 0, 2] = 65000.0
    x[0, 0, 2, 1::2] = 1e37
    x[0, 0, 3] = 65503.99
    x[0, 0, 3, 0] = 3.3e38
    x[0, 0, 4] = -65503.0
    x[0, 0, 4, 5] = -3e38
    x[0, 0, 5, 5], x[0, 0, 5, 6] = 3e38, -3e38
    x[0, 0, 6, 5] = 3e38
    x[0, 0, 7, 5] = -3e38
    x[0, 0, 8] = 65503.0
    x[0, 0, 8, 5] = math.inf
    x[0, 0, 9] = -65504.0
    x[0, 0, 9, 5] = -65503.0
    x[0, 0, 9, 6] = -math.inf
    x = x.to(dtype)
    _exactly(*fused_attn.quantize_kv_int4(x), x)
    pool = [torch.zeros(1, 1, 12, w, dtype=t, device="cuda") for w, t in ((d // 2, torch.uint8), (2, torch.float16))]
    twin = [t.clone() for t in pool]
    fused_attn.append_kv_int4(x, x, *pool, *twin, torch.zeros(1, dtype=torch.int32, device="cuda"))
    _exactly(*pool, x), _exactly(*twin, x)


@pytest.mark.parametrize("int4", [False, True])
def test_scored_of_an_empty_batch(int4):
    announce(f"scored empty batch int4={int4}")
    q = torch.zeros(0, 4, 1, 64, device="cuda").half()
    if int4:
        k, extra = torch.zeros(0, 2, 9, 32, dtype=torch.uint8, device="cuda"), torch.zeros(0, 2, 9, 2, device="cuda").half()
        extra = dict(k_scale=extra, v_scale=extra)
    else:
        k, extra = torch.zeros(0, 2, 9, 64, device="cuda").half(), {}
    o, w = fused_attn.attention_scored(q, k, k, **extra)
    assert o.shape == q.shape and w.shape == (0, 2, 9) and w.dtype == torch.float32
    # no queries and no keys
    o, w = fused_attn.attention_scored(torch.zeros(2, 4, 0, 64, device="cuda").half(), torch.zeros(2, 2, 0, 64, device="cuda").half(),
                                       torch.zeros(2, 2, 0, 64, device="cuda").half())
    assert o.shape == (2, 4, 0, 64) and w.shape == (2, 2, 0)


@pytest.mark.parametrize("d", [16, 32, 96])
@pytest.mark.parametrize("paged", [False, True])
def test_append_at_other_head_dims(d, paged):
    """The torch form, as for the writer and the reader."""
    announce(f"int4 append d={d} paged={paged}")
    b, hkv, new, page = 4, 3, 2, 16
    lens = torch.tensor([0, 15, 31, -1], dtype=torch.int32, device="cuda")
    k, v = rows((b, hkv, new, d), torch.float16, 1), rows((b, hkv, new, d), torch.float16, 2)
    shape = (9, hkv, page) if paged else (b, hkv, 2 * page)
    caches = [torch.zeros(*shape, w, dtype=t, device="cuda") for w, t in
              ((d // 2, torch.uint8), (2, torch.float16)) * 2]
    bt = torch.tensor([[8, 1], [0, 2], [3, 4], [5, 6]], dtype=torch.int32, device="cuda") if paged else None
    want = [t.cpu() for t in caches]
    fused_attn.append_kv_int4(k.cpu(), v.cpu(), *want, lens.cpu(), block_table=None if bt is None else bt.cpu())
    fused_attn.append_kv_int4(k, v, *caches, lens, block_table=bt)
    for g, w in zip(caches, want):
        assert torch.equal(g.cpu(), w) and g.any()


def test_evict_into_two_halves_of_one_buffer():
    announce("evict interleaved out")
    b, h, n, keep = 2, 3, 200, 50
    scores = torch.rand(b, h, n, device="cuda", generator=gen(1))
    k, v = (torch.randn(b, h, n, 64, device="cuda", generator=gen(i)).half() for i in (2, 3))
    both = torch.zeros(b, h, keep + 3, 2, 64, device="cuda").half()
    want, _, index, _ = fused_attn.evict_kv(scores, (k, v), keep, 5)
    got = fused_attn.evict_kv(scores, (k, v), keep, 5, out=(both[..., 0, :], both[..., 1, :]))
    for i in range(2):
        assert torch.equal(both[:, :, :keep, i], want[i])
    assert not both[:, :, keep:].any() and torch.equal(got[2], index)
