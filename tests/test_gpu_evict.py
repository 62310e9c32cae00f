"""Scored attention and eviction on the GPU, against the float64 oracle."""
import math

import pytest
import torch

import fused_attn
from cache_helpers import cache, check, garbage_behind, gen, oracle, rows
from helpers import announce

pytestmark = pytest.mark.gpu


def _case(int4, b, hkv, n, d, dtype, lens=None):
    """(k, v, scale arguments, their values in float64, pairs)"""
    if int4:
        (k, ks), (v, vs) = cache(b, hkv, n, d, 1), cache(b, hkv, n, d, 2)
        if lens is not None:
            garbage_behind(k, ks, lens), garbage_behind(v, vs, lens)
        return k, v, dict(k_scale=ks, v_scale=vs), oracle.values(k, ks), oracle.values(v, vs), (ks, vs)
    k, v = rows((b, hkv, n, d), dtype, 1), rows((b, hkv, n, d), dtype, 2)
    if lens is not None:
        garbage_behind(k, None, lens), garbage_behind(v, None, lens)
    return k, v, {}, k.double(), v.double(), None


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nk", [1, 32, 45, 600])
@pytest.mark.parametrize("hq,hkv,nq,causal", [(4, 4, 1, True), (8, 2, 1, False), (8, 2, 6, True), (4, 2, 33, True)])
def test_scored(int4, dtype, d, nk, hq, hkv, nq, causal):
    announce(f"scored int4={int4} {dtype} d={d} nk={nk} hq={hq} hkv={hkv} nq={nq} causal={causal}")
    q = torch.randn(2, hq, nq, d, device="cuda", generator=gen(nk)).to(dtype)
    k, v, extra, kv, vv, pairs = _case(int4, 2, hkv, nk, d, dtype)
    want = oracle.attention(q, kv, vv, causal)
    before = torch.rand(2, hkv, nk, device="cuda", generator=gen(1))
    for split, scores in ((None, None), (64, before)):
        kept = None if scores is None else scores.clone()
        got, w = fused_attn.attention_scored(q, k, v, scores=scores, causal=causal, split_len=split, **extra)
        assert w.dtype == torch.float32 and w.shape == (2, hkv, nk)
        check(got, *want, q, kv, vv, pairs, got_w=w, before=scores)
        assert scores is None or torch.equal(scores, kept)


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("nq,causal", [(1, True), (5, True), (5, False)])
def test_scored_lengths(int4, nq, causal):
    announce(f"scored lengths int4={int4} nq={nq} causal={causal}")
    lens = [0, 1, 500, 131, -3, 900, 3]
    q = torch.randn(7, 8, nq, 128, device="cuda", generator=gen(1)).bfloat16()
    k, v, extra, kv, vv, pairs = _case(int4, 7, 2, 500, 128, torch.bfloat16, lens)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = oracle.attention(q, kv, vv, causal, lens=lens)
    before = torch.rand(7, 2, 600, device="cuda", generator=gen(1))[..., 50:550]  # rows of a larger buffer
    for split in (None, 64):
        got, w = fused_attn.attention_scored(q, k, v, scores=before, causal=causal, seqlens_k=sl, split_len=split, **extra)
        check(got, *want, q, kv.nan_to_num(), vv.nan_to_num(), pairs, got_w=w, before=before)
        for i, n in enumerate(lens):
            assert torch.equal(w[i, :, max(n, 0):], before[i, :, max(n, 0):])


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("split", [64, 1024])  # 33 and 3 partitions
@pytest.mark.parametrize("hq,nq", [(4, 1), (32, 1), (8, 25), (8, 130)])  # 2, 16, 100 and 520 rows
def test_scored_many_rows_and_partitions(int4, split, hq, nq):
    announce(f"scored rows int4={int4} split={split} hq={hq} nq={nq}")
    lens = [2100, 1111]
    q = torch.randn(2, hq, nq, 64, device="cuda", generator=gen(1)).half()
    k, v, extra, kv, vv, pairs = _case(int4, 2, 2, 2100, 64, torch.float16, lens)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = oracle.attention(q, kv, vv, True, lens=lens)
    got, w = fused_attn.attention_scored(q, k, v, causal=True, seqlens_k=sl, split_len=split, **extra)
    check(got, *want, q, kv.nan_to_num(), vv.nan_to_num(), pairs, got_w=w)


@pytest.mark.parametrize("int4", [False, True])
def test_scored_scales_and_ragged_layouts(int4):
    announce(f"scored layouts int4={int4}")
    q = torch.randn(2, 3, 4, 64, device="cuda", generator=gen(1)).half().transpose(1, 2)
    k, v, extra, kv, vv, pairs = _case(int4, 2, 2, 77, 64, torch.float16)
    k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    for scale in (0.0, -0.5, 2.0):
        got, w = fused_attn.attention_scored(q, k, v, causal=True, scale=scale, **extra)
        check(got, *oracle.attention(q, kv, vv, True, scale), q, kv, vv, pairs, scale, got_w=w)
    one = {x: t[:1] for x, t in extra.items()}
    got, w = fused_attn.attention_scored(q, k[:1], v[:1], causal=True, **one)
    check(got, *oracle.attention(q, kv[:1], vv[:1], True), q, kv[:1], vv[:1], pairs, got_w=w)


def test_scored_sums_and_precision():
    """The weights of a row sum to 1, and to fp32's precision as a whole: the rounding of 3000 scores is random, about
    sqrt(D) half-steps of partial sums below 16 (2^-24 * 11 * 16 = 1e-5 of a weight)."""
    announce("scored precision")
    for int4 in (False, True):
        q = torch.randn(2, 8, 1, 128, device="cuda", generator=gen(1)).bfloat16()
        k, v, extra, kv, vv, _ = _case(int4, 2, 2, 3000, 128, torch.bfloat16)
        _, w = fused_attn.attention_scored(q, k, v, **extra)
        want = oracle.attention(q, kv, vv)[2]
        assert (w.double().sum(-1) - 4).abs().max() < 1e-4
        assert ((w.double() - want).norm() / want.norm()) < 2e-5


def test_scored_without_keys_or_queries():
    announce("scored empty")
    q = torch.randn(2, 4, 1, 64, device="cuda").half()
    none = torch.zeros(2, 2, 0, 64, device="cuda").half()
    o, w = fused_attn.attention_scored(q, none, none)
    assert (o == 0).all() and w.shape == (2, 2, 0)
    kv = torch.randn(2, 2, 9, 64, device="cuda").half()
    before = torch.rand(2, 2, 9, device="cuda")
    o, w = fused_attn.attention_scored(q[:, :, :0], kv, kv, scores=before)
    assert o.shape == (2, 4, 0, 64) and torch.equal(w, before) and w is not before
    assert (fused_attn.attention_scored(q[:, :, :0], kv, kv)[1] == 0).all()


def _scores(b, h, n, kind, seed=0):
    g = gen(seed)
    if kind == "weights":  # few keys hold most, some hold none
        return torch.exp(3 * torch.randn(b, h, n, device="cuda", generator=g)) * (torch.rand(b, h, n, device="cuda", generator=g) > 0.2)
    if kind == "ties":
        return torch.randint(-3, 4, (b, h, n), device="cuda", generator=g).float() * 0.25
    if kind == "equal":
        return torch.full((b, h, n), -0.0, device="cuda")
    s = torch.randn(b, h, n, device="cuda", generator=g)  # every kind of float
    u = torch.rand(b, h, n, device="cuda", generator=g)
    s = torch.where(u < 0.1, torch.full_like(s, math.nan), s)
    s = torch.where((u > 0.1) & (u < 0.2), torch.full_like(s, math.inf), s)
    s = torch.where((u > 0.2) & (u < 0.3), torch.full_like(s, -math.inf), s)
    return torch.where((u > 0.3) & (u < 0.4), s * 1e-42, s)


@pytest.mark.parametrize("n,keep,recent", [(33000, 9000, 500), (70001, 35000, 0), (150000, 149000, 7)])
@pytest.mark.parametrize("kind", ["weights", "ties", "any"])
def test_evict_many_keys(kind, n, keep, recent):
    """More candidates than are held in registers at a time; ties that fill the whole threshold digit."""
    announce(f"evict many {kind} n={n}")
    scores = _scores(1, 2, n, kind, n)
    _, s2, index, _ = fused_attn.evict_kv(scores, [], keep, recent)
    s = scores.cpu().nan_to_num(nan=math.inf, posinf=3e38) + 0.0  # (NaN above +inf, -0 as 0)
    s = torch.where(scores.cpu().isnan(), torch.full_like(s, math.inf), s)
    old = n - recent
    best = torch.sort(s[..., :old], dim=-1, descending=True, stable=True).indices[..., :keep - recent]
    want = torch.cat([torch.sort(best, dim=-1).values, torch.arange(old, n).expand(1, 2, recent)], -1)
    assert torch.equal(index.cpu().long(), want)
    assert torch.equal(s2.cpu().view(torch.int32), scores.cpu().gather(-1, want).view(torch.int32))


@pytest.mark.parametrize("lens", [[20000, 8191, 8193, 0, 16384], [16385, 20001, 101, 100, 99]])
@pytest.mark.parametrize("kind", ["weights", "equal"])
def test_evict_many_keys_of_other_lengths(kind, lens):
    """Sequences whose candidates end in an early workgroup's range, beside ones that all stay."""
    announce(f"evict many lengths {kind} {lens}")
    b, n, keep, recent = len(lens), 20001, 100, 9
    scores = _scores(b, 2, n, kind, 3)
    k = torch.randn(b, 2, n, 64, device="cuda", generator=gen(4)).half()
    (k2,), s2, index, left = fused_attn.evict_kv(scores, (k,), keep, recent, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert left.tolist() == [min(x, keep) for x in lens]
    for i in range(b):
        for j in range(2):
            at = oracle.kept(scores[i, j].cpu().numpy(), lens[i], keep, recent)
            assert index[i, j].tolist() == at + [-1] * (keep - len(at))
            assert torch.equal(k2[i, j, :len(at)], k[i, j, at]) and not k2[i, j, len(at):].any()
            assert torch.equal(s2[i, j, :len(at)], scores[i, j, at]) and not s2[i, j, len(at):].any()


def test_evict_other_types():
    announce("evict types")
    scores = _scores(2, 2, 50, "weights")
    caches = [torch.randn(2, 2, 50, 16, device="cuda").to(torch.float8_e4m3fn), torch.rand(2, 2, 50, device="cuda") > 0.5,
              torch.randn(2, 2, 50, 3, device="cuda", dtype=torch.complex64)]
    got, _, index, _ = fused_attn.evict_kv(scores, caches, 20)
    for g, c in zip(got, caches):
        at = index.long()
        for i in range(2):
            for j in range(2):
                assert torch.equal(g[i, j].view(torch.uint8), c[i, j].view(torch.uint8)[at[i, j]])


@pytest.mark.parametrize("kind", ["weights", "ties", "equal", "any"])
@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (1, 0, 0), (7, 3, 1), (1000, 999, 0), (1000, 1, 0), (1000, 300, 300),
                                           (4099, 2000, 77), (9001, 4500, 1000)])
def test_evict(kind, n, keep, recent):
    announce(f"evict {kind} n={n} keep={keep} recent={recent}")
    b, h = 2, 3
    scores = _scores(b, h, n, kind, n)
    k = torch.randn(b, h, n, 64, device="cuda", generator=gen(1)).half()
    (k2,), s2, index, left = fused_attn.evict_kv(scores, (k,), keep, recent)
    assert left.tolist() == [min(n, keep)] * b and index.shape == (b, h, min(n, keep))
    for i in range(b):
        for j in range(h):
            at = oracle.kept(scores[i, j].cpu().numpy(), n, keep, recent)
            assert index[i, j].tolist() == at
            assert torch.equal(k2[i, j], k[i, j, at])
            assert torch.equal(s2[i, j].view(torch.int32), scores[i, j, at].contiguous().view(torch.int32))


@pytest.mark.parametrize("lens", [[700, 0, 3, 350, -1, 5000], None])
def test_evict_lengths_types_and_layouts(lens):
    announce(f"evict lengths {lens}")
    b, h, n, keep, recent = 6, 2, 700, 100, 10
    scores = _scores(b, h, 720, "weights")[..., 13:713]  # rows that start at any float
    caches = [torch.randint(0, 255, (b, h, n, 64), dtype=torch.uint8, device="cuda"),
              torch.randn(b, h, n, 2, device="cuda").half(),
              torch.randn(b, n, h, 128, device="cuda").bfloat16().transpose(1, 2),
              torch.randn(b, h, n, 5, 3, device="cuda"),
              torch.randn(b, h, n, device="cuda").double(),
              torch.randint(0, 255, (b, h, n, 7), dtype=torch.uint8, device="cuda"),
              torch.randn(1, h, n, 4, device="cuda").expand(b, h, n, 4),
              torch.randn(b, h, n, 4, 6, device="cuda").transpose(-1, -2)]
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got, s2, index, left = fused_attn.evict_kv(scores, caches, keep, recent, sl)
    for i in range(b):
        m = n if lens is None else min(max(lens[i], 0), n)
        assert left[i] == min(m, keep)
        for j in range(h):
            at = oracle.kept(scores[i, j].cpu().numpy(), m, keep, recent)
            assert index[i, j].tolist() == at + [-1] * (keep - len(at))
            for g, c in zip((*got, s2), (*caches, scores)):
                assert torch.equal(g[i, j, :len(at)], c[i, j, at]) and (g[i, j, len(at):] == 0).all()


def test_evict_out_and_nothing_to_move():
    announce("evict out")
    scores, k = _scores(2, 2, 300, "weights"), torch.randn(2, 2, 300, 128, device="cuda").half()
    room = torch.full((2, 150, 2, 128), 5.0, device="cuda").half().transpose(1, 2)
    (got,), _, index, _ = fused_attn.evict_kv(scores, [k], 120, 20, out=[room])
    want = fused_attn.evict_kv(scores, [k], 120, 20)[0][0]
    assert got is room and torch.equal(room[:, :, :120], want) and (room[:, :, 120:] == 5).all()
    none, s2, index, left = fused_attn.evict_kv(scores, [], 120, 20)
    assert none == [] and s2.shape == index.shape == (2, 2, 120)
    (e,), s2, index, left = fused_attn.evict_kv(scores, [k], 0)
    assert e.shape == (2, 2, 0, 128) and left.tolist() == [0, 0]
    (e,), s2, index, left = fused_attn.evict_kv(scores[:, :, :0], [k[:, :, :0]], 5)
    assert e.shape == (2, 2, 0, 128) and left.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="share memory"):
        fused_attn.evict_kv(scores, [k], 120, out=[k[:, :, :150]])


def test_evict_long_cache():
    """Row offsets past 2^31 bytes and 2^31 elements."""
    announce("evict long")
    n = 9_000_000
    k = torch.zeros(1, 1, n, 256, dtype=torch.float16, device="cuda")  # 4.6 GB
    scores = torch.zeros(1, 1, n, device="cuda")
    at = torch.tensor([3, n // 2, n - 9, n - 2], device="cuda")
    scores[0, 0, at] = torch.tensor([1.0, 3.0, 2.0, 4.0], device="cuda")
    k[0, 0, at, 0] = torch.tensor([1.0, 3.0, 2.0, 4.0], device="cuda").half()
    (k2,), s2, index, _ = fused_attn.evict_kv(scores, [k], 5, 1)
    assert index.flatten().tolist() == [*at.tolist(), n - 1] and k2[0, 0, :, 0].tolist() == [1, 3, 2, 4, 0]


@pytest.mark.parametrize("int4", [False, True])
def test_score_and_evict_together(int4):
    """Decode steps that score a cache, an eviction, and more steps over what is left."""
    announce(f"score and evict int4={int4}")
    b, hq, hkv, n, d, keep, recent = 2, 8, 2, 300, 128, 100, 30
    lens = [300, 260]
    k, v, extra, kv, vv, pairs = _case(int4, b, hkv, n, d, torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scores, total = None, torch.zeros(b, hkv, n, dtype=torch.float64, device="cuda")
    for step in range(3):
        q = torch.randn(b, hq, 1, d, device="cuda", generator=gen(step)).bfloat16()
        _, scores = fused_attn.attention_scored(q, k, v, scores=scores, causal=True, seqlens_k=sl, **extra)
        total += oracle.attention(q, kv, vv, True, lens=lens)[2]
    assert (scores.double() - total).abs().max() < 1e-4
    caches = [k, v, *extra.values()]
    caches, scores, index, sl = fused_attn.evict_kv(scores, caches, keep, recent, sl)
    assert sl.tolist() == [keep, keep]
    for i in range(b):  # what stays has the highest true scores, up to the error of the sums
        for j in range(hkv):
            gone = [x for x in range(lens[i]) if x not in set(index[i, j].tolist())]
            old = [x for x in index[i, j].tolist() if x < lens[i] - recent]
            assert total[i, j, old].min() >= total[i, j, gone].max() - 2e-4
    extra = dict(zip(extra, caches[2:]))
    q = torch.randn(b, hq, 1, d, device="cuda", generator=gen(9)).bfloat16()
    got, _ = fused_attn.attention_scored(q, caches[0], caches[1], scores=scores, causal=True, seqlens_k=sl, **extra)
    at = index.long()[..., None].expand(b, hkv, keep, d)
    k2, v2 = kv.gather(2, at), vv.gather(2, at)
    check(got, *oracle.attention(q, k2, v2, True), q, k2, v2, pairs)


def test_evict_many_keys_in_a_graph_and_twice_at_once():
    announce("evict many graph")
    n, keep = 30000, 7000
    scores = [_scores(1, 2, n, "weights", i) for i in range(2)]
    want = [fused_attn.evict_kv(s, [], keep, 100)[2] for s in scores]
    graphs, got = [], []
    for s in scores:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(fused_attn.evict_kv(s, [], keep, 100)[2])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in scores]
    torch.cuda.synchronize()
    for _ in range(4):
        for x in got:
            x.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for x, w in zip(got, want):
            assert torch.equal(x, w)
        torch.ones(1000, device="cuda").sum().item()


def test_scored_and_evict_in_a_graph():
    announce("score and evict graph")
    b, hq, hkv, n, d = 2, 4, 2, 600, 64
    q = torch.randn(b, hq, 1, d, device="cuda", generator=gen(1)).half()
    k, v = rows((b, hkv, n, d), torch.float16, 1), rows((b, hkv, n, d), torch.float16, 2)
    sl = torch.tensor([600, 555], dtype=torch.int32, device="cuda")
    before = torch.rand(b, hkv, n, device="cuda", generator=gen(2))

    def step():
        o, s = fused_attn.attention_scored(q, k, v, scores=before, causal=True, seqlens_k=sl)
        return o, s, fused_attn.evict_kv(s, (k, v), 200, 50, sl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s, (caches, s2, index, left) = step()
    for i in range(4):
        q.normal_(generator=gen(20 + i))
        before.uniform_(generator=gen(30 + i))
        eo, es, (ecaches, es2, eindex, eleft) = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip((o, s, *caches, s2, index, left), (eo, es, *ecaches, es2, eindex, eleft)):
            assert torch.equal(a, c), i
