"""The 4-bit cache on the GPU: writer and reader bit for bit against the definition, attention (dense and paged) against
the float64 oracle on the rows that the codes stand for."""
import math

import numpy as np
import pytest
import torch

import fused_attn
from cache_helpers import cache, check, garbage_behind, gen, oracle, rows
from helpers import announce

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _exactly(codes, pairs, x):
    code, scale, zero = oracle.encode(x)
    want = torch.from_numpy(np.stack([scale, zero], -1))
    assert torch.equal(codes.cpu(), torch.from_numpy(oracle.pack(code)))
    got, want = pairs.cpu().float(), want.float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 17), (1, 8, 1000), (3, 2, 129)])
def test_writer_and_reader(dtype, d, shape):
    announce(f"int4 rows {dtype} d={d} {shape}")
    x = rows((*shape, d), dtype, sum(shape))
    codes, pairs = fused_attn.quantize_kv_int4(x)
    _exactly(codes, pairs, x)
    for out in DTYPES:
        assert torch.equal(fused_attn.dequantize_kv_int4(codes, pairs, out), oracle.values(codes, pairs).float().to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_writer_at_ties_and_at_the_edges_of_its_types(dtype):
    announce(f"int4 edges {dtype}")
    x = torch.randn(1, 1, 16, 64, device="cuda", generator=gen(1))
    x[0, 0, 0] = torch.arange(64, device="cuda") % 31 * 0.5  # every step and every half step
    x[0, 0, 1] = -1.5
    x[0, 0, 2] = 0.0
    x[0, 0, 3] *= 1e-6
    x[0, 0, 4] *= 1e-7
    x[0, 0, 5] = x[0, 0, 5] * 3e4
    x[0, 0, 6, 5] = math.inf
    x[0, 0, 7, 6] = -math.inf
    x[0, 0, 8, 7] = math.nan
    x[0, 0, 9] = math.inf
    x[0, 0, 10] += 1000.0
    x[0, 0, 11, ::2] = -0.0
    x[0, 0, 12] *= 1e30 if dtype != torch.float16 else 1.0
    x = x.to(dtype)
    codes, pairs = fused_attn.quantize_kv_int4(x)
    _exactly(codes, pairs, x)
    # (a zero scale times any code is 0, so the value is zero + 0)
    got, want = fused_attn.dequantize_kv_int4(codes, pairs).double(), oracle.values(codes, pairs).float().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_writer_and_reader_views():
    announce("int4 views")
    x = rows((2, 50, 3, 128), torch.bfloat16, 3).transpose(1, 2)  # a [B, N, H, D] projection
    codes, pairs = fused_attn.quantize_kv_int4(x)
    _exactly(codes, pairs, x.contiguous())
    odd = rows((2, 3, 50, 136), torch.float16, 4)[..., 3:131]  # unaligned rows: copied first
    _exactly(*fused_attn.quantize_kv_int4(odd), odd.contiguous())
    # into a slice of a larger cache, and back out of it
    whole = torch.full((2, 3, 80, 64), 9, dtype=torch.uint8, device="cuda"), \
        torch.full((2, 3, 80, 2), 9.0, dtype=torch.float16, device="cuda")
    fused_attn.quantize_kv_int4(x, out=tuple(t[:, :, 20:70] for t in whole))
    assert torch.equal(whole[0][:, :, 20:70], codes) and torch.equal(whole[1][:, :, 20:70], pairs)
    for t in whole:
        assert (t[:, :, :20] == 9).all() and (t[:, :, 70:] == 9).all()
    got = fused_attn.dequantize_kv_int4(whole[0][:, :, 20:70], whole[1][:, :, 20:70], torch.bfloat16)
    assert torch.equal(got, fused_attn.dequantize_kv_int4(codes, pairs, torch.bfloat16))
    # a [B, N, H, *] cache
    turned = torch.zeros(2, 50, 3, 64, dtype=torch.uint8, device="cuda"), torch.zeros(2, 50, 3, 2, device="cuda").half()
    fused_attn.quantize_kv_int4(x, out=tuple(t.transpose(1, 2) for t in turned))
    assert torch.equal(turned[0].transpose(1, 2), codes) and torch.equal(turned[1].transpose(1, 2), pairs)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("paged", [False, True])
def test_append(d, paged):
    announce(f"int4 append d={d} paged={paged}")
    b, hkv, cap, new, page = 5, 3, 64, 3, 16
    lens = [0, 5, 15, 62, -1]  # 62: one token has no room; -1: the first token has no place
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = rows((b, hkv, new, d), torch.bfloat16, 1), rows((b, new, hkv, d), torch.bfloat16, 2).transpose(1, 2)
    shape = (b * 4 + 2, hkv, page) if paged else (b, hkv, cap)
    caches = [torch.full((*shape, w), 3, dtype=t, device="cuda") for w, t in
              ((d // 2, torch.uint8), (2, torch.float16), (d // 2, torch.uint8), (2, torch.float16))]
    bt = None
    if paged:
        bt = torch.randperm(b * 4 + 2, device="cuda", generator=gen(3))[:b * 4].view(b, 4).to(torch.int32)
        bt[1, 0] = 99  # outside the pool
    want = [t.clone() for t in caches]
    for x, c, s in ((k, want[0], want[1]), (v, want[2], want[3])):
        codes, pairs = fused_attn.quantize_kv_int4(x)
        for i, n in enumerate(lens):
            for j in range(new):
                if not 0 <= n + j < cap or (paged and i == 1):
                    continue
                at, pos = (int(bt[i, (n + j) // page]), (n + j) % page) if paged else (i, n + j)
                c[at, :, pos], s[at, :, pos] = codes[i, :, j], pairs[i, :, j]
    fused_attn.append_kv_int4(k, v, *caches, sl, block_table=bt)
    for got, w in zip(caches, want):
        assert torch.equal(got, w)
    assert sl.tolist() == lens


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nk", [1, 31, 33, 128, 1000])
@pytest.mark.parametrize("hq,hkv,nq,causal", [(4, 4, 1, False), (8, 2, 3, True), (8, 1, 5, True), (4, 2, 40, True)])
def test_attention(dtype, d, nk, hq, hkv, nq, causal):
    announce(f"int4 attention {dtype} d={d} nk={nk} hq={hq} hkv={hkv} nq={nq} causal={causal}")
    q = torch.randn(2, hq, nq, d, device="cuda", generator=gen(nk)).to(dtype)
    (k4, ks), (v4, vs) = cache(2, hkv, nk, d, 1), cache(2, hkv, nk, d, 2)
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    want = oracle.attention(q, k, v, causal)
    for split in (None, 64):
        got, lse = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=causal, split_len=split, return_lse=True)
        check(got, *want, q, k, v, (ks, vs), got_lse=lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 6, 30])  # 4, 24 and 120 rows
@pytest.mark.parametrize("split", [64, 128, 1024])  # 40, 20 and 3 partitions: the merges of many and of few
def test_attention_many_partitions(d, nq, split):
    announce(f"int4 partitions d={d} nq={nq} split={split}")
    lens = [2500, 1300, 0]
    q = torch.randn(3, 8, nq, d, device="cuda", generator=gen(1)).half()
    (k4, ks), (v4, vs) = cache(3, 2, 2500, d, 1), cache(3, 2, 2500, d, 2)
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    for sl in (None, torch.tensor(lens, dtype=torch.int32, device="cuda")):
        want = oracle.attention(q, k, v, True, lens=None if sl is None else lens)
        got, lse = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=True, seqlens_k=sl, split_len=split, return_lse=True)
        check(got, *want, q, k, v, (ks, vs), got_lse=lse)


def test_attention_of_infinite_and_nan_keys():
    """A score of -inf (finite operands whose product is not) weighs nothing; a NaN key makes the rows that see it NaN."""
    announce("int4 infinite scores")
    q = torch.full((1, 2, 2, 64), 3e38, device="cuda").bfloat16()
    k = torch.randn(1, 1, 70, 64, device="cuda", generator=gen(1)) * 1e-38
    k[0, 0, 5], k[0, 0, 40] = -6e4, -6e4
    k4, ks = fused_attn.quantize_kv_int4(k)
    v4, vs = cache(1, 1, 70, 64, 2)
    got = fused_attn.attention_int4(q, k4, ks, v4, vs, scale=1e-3)
    keep = [j for j in range(70) if j not in (5, 40)]
    want = fused_attn.attention_int4(q, k4[:, :, keep], ks[:, :, keep], v4[:, :, keep], vs[:, :, keep], scale=1e-3)
    assert torch.isfinite(got).all() and (got.float() - want.float()).abs().max() < 0.05
    ks = ks.clone()
    ks[0, 0, 69] = math.nan
    got = fused_attn.attention_int4(q.clamp(max=1.0), k4, ks, v4, vs)
    assert torch.isnan(got).all()
    got = fused_attn.attention_int4(q.clamp(max=1.0), k4, ks, v4, vs, seqlens_k=torch.tensor([69], device="cuda").int())
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("lens", [[0, 1, 700, 64], [-5, 9999, 33, 2]])
@pytest.mark.parametrize("nq,causal", [(1, True), (4, True), (4, False), (20, True)])
def test_attention_lengths(lens, nq, causal):
    announce(f"int4 lengths {lens} nq={nq} causal={causal}")
    q = torch.randn(4, 8, nq, 128, device="cuda", generator=gen(1)).bfloat16()
    (k4, ks), (v4, vs) = cache(4, 2, 700, 128, 1), cache(4, 2, 700, 128, 2)
    garbage_behind(k4, ks, lens), garbage_behind(v4, vs, lens)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    want = oracle.attention(q, k, v, causal, lens=lens)
    for split in (None, 64, 320):
        got, lse = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=causal, seqlens_k=sl, split_len=split,
                                             return_lse=True)
        check(got, *want, q, k, v, (ks, vs), got_lse=lse)


@pytest.mark.parametrize("scale", [0.0, -0.3, 0.7, 4.0])
def test_attention_scales(scale):
    announce(f"int4 scale {scale}")
    q = torch.randn(2, 4, 2, 64, device="cuda", generator=gen(1)).half()
    (k4, ks), (v4, vs) = cache(2, 2, 300, 64, 1), cache(2, 2, 300, 64, 2)
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    check(fused_attn.attention_int4(q, k4, ks, v4, vs, True, scale), *oracle.attention(q, k, v, True, scale), q, k, v,
          (ks, vs), scale)


def test_attention_magnitudes():
    """V rows of magnitudes 1e-4 to 1e3 next to each other, K rows far from zero."""
    announce("int4 magnitudes")
    d = 128
    q = torch.randn(1, 4, 1, d, device="cuda", generator=gen(1)).half()
    mags = torch.tensor([1e-4, 1.0, 1e3, 0.05], device="cuda").repeat(64)[None, None, :, None]
    k4, ks = fused_attn.quantize_kv_int4(rows((1, 1, 256, d), torch.float32, 1).cpu() + 20)
    v4, vs = fused_attn.quantize_kv_int4((rows((1, 1, 256, d), torch.float32, 2) * mags).cpu())
    k4, ks, v4, vs = (t.cuda() for t in (k4, ks, v4, vs))
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    check(fused_attn.attention_int4(q, k4, ks, v4, vs), *oracle.attention(q, k, v), q, k, v, (ks, vs))
    small = v[:, :, 0::4], v4[:, :, 0::4], vs[:, :, 0::4]  # the 1e-4 rows alone: fp16 pairs down to subnormal ones
    check(fused_attn.attention_int4(q, k4[:, :, 0::4], ks[:, :, 0::4], small[1], small[2]),
          *oracle.attention(q, k[:, :, 0::4], small[0]), q, k[:, :, 0::4], small[0], (ks[:, :, 0::4], small[2]))


def test_attention_views_and_shared_batch():
    announce("int4 views")
    b, hkv, n, d = 3, 2, 150, 128
    q = torch.randn(b, 5, 4, d, device="cuda", generator=gen(1)).bfloat16().transpose(1, 2)  # [B, N, H, D]
    (k4, ks), (v4, vs) = cache(b, hkv, n, d, 1), cache(b, hkv, n, d, 2)
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    want = oracle.attention(q, k, v, True)
    room = torch.zeros(b, hkv, n + 37, d // 2, dtype=torch.uint8, device="cuda")
    room[:, :, :n] = k4
    turned = v4.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(b, hkv, n, 3, dtype=torch.float16, device="cuda")  # pairs on odd halves: copied first
    odd[..., 1:] = ks
    got = fused_attn.attention_int4(q, room[:, :, :n], odd[..., 1:], turned, vs.transpose(1, 2).contiguous().transpose(1, 2),
                                    causal=True)
    check(got, *want, q, k, v, (ks, vs))
    one = fused_attn.attention_int4(q, k4[1:2], ks[1:2], v4[1:2], vs[1:2], causal=True)
    check(one, *oracle.attention(q, k[1:2], v[1:2], True), q, k[1:2], v[1:2], (ks, vs))


def test_attention_without_keys_or_queries():
    announce("int4 empty")
    q = torch.randn(2, 4, 1, 64, device="cuda").half()
    none = torch.zeros(2, 2, 0, 32, dtype=torch.uint8, device="cuda"), torch.zeros(2, 2, 0, 2, device="cuda").half()
    got, lse = fused_attn.attention_int4(q, *none, *none, return_lse=True)
    assert (got == 0).all() and torch.isneginf(lse).all()
    k4, ks = cache(2, 2, 8, 64)
    assert fused_attn.attention_int4(q[:, :, :0], k4, ks, k4, ks).shape == (2, 4, 0, 64)
    assert fused_attn.attention_int4(q[:0], k4[:0], ks[:0], k4[:0], ks[:0]).shape == (0, 4, 1, 64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("nq", [1, 9])
def test_paged(dtype, d, page, nq):
    announce(f"int4 paged {dtype} d={d} page={page} nq={nq}")
    lens = [500, 0, 257, 1]
    q = torch.randn(4, 8, nq, d, device="cuda", generator=gen(1)).to(dtype)
    (k4, ks), (v4, vs) = cache(4, 2, 500, d, 1), cache(4, 2, 500, d, 2)
    garbage_behind(k4, ks, lens), garbage_behind(v4, vs, lens)
    kp, vp, ksp, vsp, bt, sl = fused_attn.paged_from_dense_int4(k4, ks, v4, vs, page, lens, extra_pages=2,
                                                                generator=torch.Generator().manual_seed(1))
    bt[1], bt[3, 1:] = -1, 1 << 30  # entries behind the sequences' keys are not read
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    want = oracle.attention(q, k, v, True, lens=lens)
    for split in (None, 64):
        got, lse = fused_attn.attention_paged(q, kp, vp, bt, sl, causal=True, split_len=split, return_lse=True,
                                              k_scale=ksp, v_scale=vsp)
        check(got, *want, q, k, v, (ks, vs), got_lse=lse)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp, ksp, vsp)]  # [pages, page, H, *] pools
    again = fused_attn.attention_paged(q, turned[0], turned[1], bt, sl, causal=True, max_seqlen_k=500, k_scale=turned[2],
                                       v_scale=turned[3], split_len=64)
    assert torch.equal(again, got)


def test_paged_without_keys_and_with_a_short_maximum():
    announce("int4 paged empty")
    q = torch.randn(2, 4, 1, 64, device="cuda").half()
    (k4, ks), (v4, vs) = cache(2, 2, 64, 64, 1), cache(2, 2, 64, 64, 2)
    kp, vp, ksp, vsp, bt, sl = fused_attn.paged_from_dense_int4(k4, ks, v4, vs, 16, generator=torch.Generator().manual_seed(1))
    got, lse = fused_attn.attention_paged(q, kp, vp, bt, torch.zeros_like(sl), k_scale=ksp, v_scale=vsp, return_lse=True)
    assert (got == 0).all() and torch.isneginf(lse).all()
    got = fused_attn.attention_paged(q, kp, vp, bt, sl, max_seqlen_k=40, k_scale=ksp, v_scale=vsp)  # read as 40
    want = fused_attn.attention_int4(q, k4[:, :, :40], ks[:, :, :40], v4[:, :, :40], vs[:, :, :40])
    assert (got.float() - want.float()).abs().max() < 1e-3


def test_paged_pages_outside_the_pool_are_zero_keys():
    announce("int4 pages outside the pool")
    q = torch.randn(1, 4, 1, 128, device="cuda", generator=gen(1)).half()
    (k4, ks), (v4, vs) = cache(1, 2, 96, 128, 1), cache(1, 2, 96, 128, 2)
    kp, vp, ksp, vsp, bt, sl = fused_attn.paged_from_dense_int4(k4, ks, v4, vs, 16, generator=torch.Generator().manual_seed(1))
    bt[0, 2], bt[0, 4] = -1, kp.shape[0]
    ks, vs = ks.clone(), vs.clone()
    for t in (ks, vs):
        t[:, :, 32:48] = 0
        t[:, :, 64:80] = 0
    k, v = oracle.values(k4, ks), oracle.values(v4, vs)
    check(fused_attn.attention_paged(q, kp, vp, bt, sl, k_scale=ksp, v_scale=vsp), *oracle.attention(q, k, v), q, k, v,
          (ks, vs))


def test_long_cache_beyond_32_bit_offsets():
    """Rows past 4 GiB of the codes: one key there holds all the weight."""
    announce("int4 long cache")
    b, hkv, n, d = 1, 1, 34_000_000, 256  # 4.35 GB of codes
    codes = torch.zeros(b, hkv, n, d // 2, dtype=torch.uint8, device="cuda")
    pairs = torch.zeros(b, hkv, n, 2, dtype=torch.float16, device="cuda")
    at = n - 5
    codes[0, 0, at], pairs[0, 0, at] = 0xFF, torch.tensor([1.0, 0.0])
    q = torch.ones(1, 2, 1, d, device="cuda").half()
    got = fused_attn.attention_int4(q, codes, pairs, codes, pairs)
    assert torch.equal(got, torch.full_like(got, 15.0))  # scores 240 and 0: the others weigh 2^-346


def test_decode_loop_and_graph():
    """Append, attend, append, attend, as a server does, eagerly and replayed from a graph."""
    announce("int4 decode loop")
    b, hq, hkv, d, page = 3, 8, 2, 128, 16
    q = torch.randn(b, hq, 1, d, device="cuda", generator=gen(1)).bfloat16()
    k, v = rows((b, hkv, 1, d), torch.bfloat16, 1), rows((b, hkv, 1, d), torch.bfloat16, 2)
    pools = [torch.zeros(24, hkv, page, w, dtype=t, device="cuda") for w, t in
             ((d // 2, torch.uint8), (2, torch.float16), (d // 2, torch.uint8), (2, torch.float16))]
    bt = torch.arange(24, dtype=torch.int32, device="cuda").view(b, 8)
    sl = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step():
        fused_attn.append_kv_int4(k, v, *pools, sl, block_table=bt)
        sl.add_(1)
        return fused_attn.attention_paged(q, pools[0], pools[2], bt, sl, causal=True, max_seqlen_k=8 * page,
                                          k_scale=pools[1], v_scale=pools[3])

    eager = []
    for i in range(20):
        k.normal_(generator=gen(10 + i)), v.normal_(generator=gen(50 + i))
        eager.append(step())
    for t in (*pools, sl):
        t.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in (*pools, sl):
        t.zero_()
    for i in range(20):
        k.normal_(generator=gen(10 + i)), v.normal_(generator=gen(50 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i


def test_other_stream_and_repeatable():
    announce("int4 streams")
    q = torch.randn(4, 8, 2, 64, device="cuda", generator=gen(1)).half()
    (k4, ks), (v4, vs) = cache(4, 2, 3000, 64, 1), cache(4, 2, 3000, 64, 2)
    want = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fused_attn.attention_int4(q, k4, ks, v4, vs, causal=True) for _ in range(3)]
    here = fused_attn.attention_int4(q, k4, ks, v4, vs, causal=True)  # two streams at once
    torch.cuda.synchronize()
    assert torch.equal(here, want) and all(torch.equal(g, want) for g in got)


def test_reference_backend_agrees(monkeypatch):
    announce("int4 reference backend")
    q = torch.randn(2, 4, 1, 64, device="cuda", generator=gen(1)).half()
    (k4, ks), (v4, vs) = cache(2, 2, 200, 64, 1), cache(2, 2, 200, 64, 2)
    got = fused_attn.attention_int4(q, k4, ks, v4, vs)
    monkeypatch.setenv("FUSED_ATTN_BACKEND", "reference")
    ref = fused_attn.attention_int4(q, k4, ks, v4, vs)
    assert (got.float() - ref.float()).abs().max() < 0.02


def test_refuses_mixed_devices():
    announce("int4 devices")
    q = torch.randn(2, 4, 1, 64, device="cuda").half()
    k4, ks = cache(2, 2, 8, 64)
    with pytest.raises(RuntimeError, match="must be on"):
        fused_attn.attention_int4(q, k4, ks, k4.cpu(), ks.cpu())
    with pytest.raises(RuntimeError, match="must be on"):
        fused_attn.attention_int4(q, k4, ks, k4, ks, seqlens_k=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="at most 258 pages"):
        bt = torch.zeros(2, 600, dtype=torch.int32, device="cuda")
        fused_attn.attention_paged(q, k4.repeat(1, 1, 2, 1), k4.repeat(1, 1, 2, 1), bt, torch.full((2,), 9600, device="cuda").int(),
                                   k_scale=ks.repeat(1, 1, 2, 1), v_scale=ks.repeat(1, 1, 2, 1), split_len=8192)
