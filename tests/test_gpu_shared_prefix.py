"""Attention behind shared prefixes on the GPU against attention in 64 bits, row by row at a tolerance on norms."""
import pytest
import torch

import fused_attn
from helpers import announce
from shared_helpers import Case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _lens(prefix, own):
    return [max(0, prefix + x) for x in own]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq,causal", [(1, False), (1, True), (3, True), (8, False), (17, True)])  # 28 to 476 rows a group
@pytest.mark.parametrize("page", [16, 48, 64])
def test_one_group(dtype, d, nq, causal, page):
    """A prefix that ends inside a tile and a page; requests with no key behind it, fewer keys than it, none at all."""
    announce(f"shared one group {dtype} d={d} nq={nq} causal={causal} page={page}")
    case = Case([7], [200], _lens(200, [0, 1, 37, 150, 64, -100, -200]), d=d, page=page, dtype=dtype)
    q = case.q(8, nq)
    o, lse = case.call(q, causal=causal, return_lse=True)
    case.check(o, q, causal, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 5])
def test_groups(dtype, d, nq):
    """Groups of several sizes, an empty one, a request alone, one without a prefix, one whose first request is padding."""
    announce(f"shared groups {dtype} d={d} nq={nq}")
    groups, prefixes = [3, 0, 1, 5, 40], [130, 64, 700, 0, 1000]
    lens = _lens(130, [5, 66, 300]) + _lens(700, [20]) + [1, 90, 300, 63, 64] + [0] + _lens(1000, [3 * i for i in range(39)])
    case = Case(groups, prefixes, lens, d=d, page=32, dtype=dtype)
    q = case.q(8, nq)
    case.check(case.call(q, causal=True), q, True)


def test_more_groups_than_a_wave_has_lanes():
    groups, prefixes = [1 + i % 3 for i in range(150)], [64 * (i % 4) + i for i in range(150)]
    lens = [p + 1 + 7 * i for p, c in zip(prefixes, groups) for i in range(c)]
    case = Case(groups, prefixes, lens, page=16)
    q = case.q(4, 2)
    case.check(case.call(q, causal=True), q, True)


@pytest.mark.parametrize("split", [None, 64, 192, 1024])
@pytest.mark.parametrize("hq,nq", [(2, 1), (16, 1), (6, 16), (32, 11)])  # 1 to 176 rows a request, 1 to 16 q-heads a kv-head
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_and_partitions(split, hq, nq, d):
    announce(f"shared rows hq={hq} nq={nq} d={d} split={split}")
    case = Case([11], [1500], _lens(1500, [1 + 83 * i for i in range(11)]), d=d, page=64)
    q = case.q(hq, nq)
    case.check(case.call(q, causal=True, split_len=split), q, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nq,page", [(1, 64), (1, 128), (4, 64), (9, 192)])
@pytest.mark.parametrize("split", [None, 64])
def test_fp8(dtype, d, nq, page, split):
    announce(f"shared fp8 {dtype} d={d} nq={nq} page={page} split={split}")
    lens = _lens(460, [0, 1, 300, 63, 64, 65, -300, -460, 129, 200])
    case = Case([10], [460], lens, d=d, page=page, fp8=True)
    q = case.q(8, nq, dtype)
    o, lse = case.call(q, causal=True, return_lse=True, split_len=split)
    case.check(o, q, True, lse)


@pytest.mark.parametrize("fp8", [False, True])
def test_many_rows(fp8):
    """Several row blocks a kv-head, several workgroups of keys."""
    case = Case([90], [3000], _lens(3000, [(17 * i) % 300 for i in range(90)]), d=128, page=64, fp8=fp8)
    q = case.q(16, 2)
    case.check(case.call(q, causal=True), q, True)


@pytest.mark.parametrize("fp8", [False, True])
def test_same_bits(fp8):
    """A number or a tensor for the prefix, bounds given or read, calls repeated over a workspace of NaN: the same bits.  One
    group given as such is the batch given whole."""
    case = Case([9], [320], _lens(320, [40 * i for i in range(9)]), d=128, page=64, fp8=fp8)
    q = case.q(8, 3)
    first = case.call(q, causal=True)
    case.check(first, q, True)
    junk = [torch.full((1 << s,), float("nan"), device="cuda") for s in range(10, 24)]
    del junk
    bounds = {"max_prefix_len": 320, "max_suffix_len": 320}
    for kw in ({}, bounds, {"prefix_lens": 320}, {"prefix_lens": 320, **bounds}, {"cu_groups": case.cu_groups}):
        assert torch.equal(case.call(q, causal=True, **kw), first), kw


def test_bounds_given_too_small_or_too_large():
    case = Case([6], [500], _lens(500, [10, 100, 0, 7, 300, 64]), d=64, page=16)
    q = case.q(8, 1)
    # larger bounds lay out a larger grid
    case.check(case.call(q, max_prefix_len=4000, max_suffix_len=2000), q)
    # the prefix is shared up to max_prefix_len, the rest is each request's own
    case.check(case.call(q, max_prefix_len=200, max_suffix_len=300 + 300), q)
    case.check(case.call(q, max_prefix_len=0, max_suffix_len=800), q)
    # keys past max_suffix_len are not read: at least 64 of them here, so that the bound's rounding does not reach them
    few = [min(n, 512) for n in case.lens]
    got = case.call(q, max_prefix_len=500, max_suffix_len=1)
    for i, n in enumerate(few):
        if n == case.lens[i]:
            continue
        assert not torch.equal(got[i], case.call(q)[i])
    assert torch.isfinite(got).all()


def test_views_and_scales():
    """Pools [num_pages, page_size, Hkv, D], queries [B, N, H, D], custom and negative scales, a table with more columns."""
    case = Case([5], [300], _lens(300, [9, 50, 100, 0, 1]), d=128, page=16)
    q = case.q(8, 4)
    want = case.call(q, causal=True)
    case.check(want, q, True)
    turned = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in (case.k, case.v)]
    wide = torch.full((5, case.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :case.table.shape[1]] = case.table
    got = fused_attn.attention_shared_prefix(q.transpose(1, 2).contiguous().transpose(1, 2), *turned, wide,
                                             case.seqlens, 300, causal=True)
    assert torch.equal(got, want)
    for scale in (0.3, -0.05, 0.0):
        got = case.call(q, scale=scale)
        want = fused_attn.attention_paged(q, case.k, case.v, case.table, case.seqlens, scale=scale)
        # both are within a norm tolerance of the exact result: 2^-7 covers twice the bf16 roundings of values about 1
        assert ((got.double() - want.double()).norm(dim=-1) <= 2.0 ** -6 * (1 + want.double().norm(dim=-1))).all()


def test_nan_stays_in_its_row():
    """A NaN query spoils its own rows alone; keys behind a request's own are never read (they are NaN in these pools)."""
    case = Case([6], [256], _lens(256, [5, 70, 0, 33, 128, 2]), d=128, page=64)
    q = case.q(8, 2)
    want = case.call(q, causal=True)
    q[3, 5, 1, 17] = float("nan")
    got = case.call(q, causal=True)
    assert torch.isnan(got[3, 5, 1]).all()
    got[3, 5, 1] = want[3, 5, 1]
    assert torch.equal(got, want)


def test_empty_calls():
    case = Case([3], [64], [64, 70, 65], d=64, page=16)
    q = case.q(4, 1)
    assert case.call(q[:, :, :0]).shape == (3, 4, 0, 64)
    none = fused_attn.attention_shared_prefix(q[:0], case.k, case.v, case.table[:0], case.seqlens[:0], 64)
    assert none.shape == (0, 4, 1, 64)
    o, lse = fused_attn.attention_shared_prefix(q, case.k[:0], case.v[:0], case.table, case.seqlens * 0, 64, return_lse=True)
    assert (o == 0).all() and torch.isneginf(lse).all()


def test_captured():
    """Lengths, tables and prefixes change between replays; every replay equals the eager call."""
    case = Case([4, 5], [300, 170], _lens(300, [5, 100, 0, 60]) + _lens(170, [1, 2, 90, 64, 200]), d=128, page=32)
    q = case.q(8, 1)
    bounds = {"max_prefix_len": 320, "max_suffix_len": 240}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        case.call(q, **bounds)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = case.call(q, **bounds)
    for i in range(5):
        q.copy_(torch.randn_like(q))
        case.seqlens.copy_(torch.tensor([max(0, n - 11 * i) for n in case.lens], dtype=torch.int32))
        case.prefix_lens.copy_(torch.tensor([300 - 40 * i, 170 - 13 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, case.call(q, **bounds))


def test_a_serving_run():
    """Pages taken, rows written, attention behind a shared system prompt, pages given back: a few steps as a server makes
    them, each step's output against attention over the keys as they were appended."""
    b, hq, hkv, d, page, prefix = 13, 8, 2, 128, 16, 160
    dtype, dev = torch.bfloat16, "cuda"
    g = torch.Generator(device=dev).manual_seed(3)
    pools = [torch.full((400, hkv, page, d), float("nan"), device=dev, dtype=dtype) for _ in "kv"]
    free = torch.randperm(400, device=dev, generator=g).to(torch.int32)
    left = torch.tensor([400], dtype=torch.int32, device=dev)
    table = torch.full((b, 40), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(b, dtype=torch.int32, device=dev)
    rows = lambda t: [torch.randn(t, hkv, d, device=dev, generator=g).to(dtype) for _ in "kv"]  # noqa: E731

    # the prompt is written once, by a request of its own, and every request's row starts with its pages
    one = torch.full((1, 40), -1, dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    slots, _, _, left = fused_attn.allocate_pages(one, zero, zero + prefix, free, left, page, prefix)
    prompt = rows(prefix)
    fused_attn.append_kv_paged(*prompt, *pools, slots)
    table[:, :prefix // page] = one[:, :prefix // page]
    lens += prefix
    history = [[[x] for _ in range(b)] for x in prompt]  # k, v: chunks of each request's keys

    for step in range(4):
        new = [3 + (5 * i + step) % 40 for i in range(b)] if step == 0 else [1] * b
        tokens = sum(new)
        slots, cu, lens, left = fused_attn.allocate_pages(table, lens, torch.tensor(new, dtype=torch.int32, device=dev), free,
                                                          left, page, tokens)
        k, v = rows(tokens)
        fused_attn.append_kv_paged(k, v, *pools, slots)
        cu = cu.tolist()
        for h, x in zip(history, (k, v)):
            for i in range(b):
                h[i].append(x[cu[i]:cu[i + 1]])
        q = torch.randn(b, hq, 1, d, device=dev, generator=g).to(dtype)
        got = fused_attn.attention_shared_prefix(q, *pools, table, lens, prefix, causal=True)
        want_lens = [sum(len(x) for x in history[0][i]) for i in range(b)]
        assert lens.tolist() == want_lens
        dense = [torch.zeros(b, hkv, max(want_lens), d, dtype=torch.float64, device=dev) for _ in "kv"]
        for t, h in zip(dense, history):
            for i in range(b):
                t[i, :, :want_lens[i]] = torch.cat(h[i]).transpose(0, 1).double()
        from cache_norms import check_rows
        check_rows(got, q, *dense, causal=True, lens=want_lens)
    done = torch.tensor([i % 2 == 0 for i in range(b)], device=dev)
    before = int(left)
    own = sum(-(-n // page) - prefix // page for i, n in enumerate(want_lens) if i % 2 == 0)
    keep = torch.full((b,), prefix, dtype=torch.int32, device=dev)
    lens, left = fused_attn.release_pages(table, lens, done, free, left, page, keep_lens=keep)
    assert int(left) == before + own and len(set(free[:int(left)].tolist())) == int(left)
    assert lens.tolist() == [0 if i % 2 == 0 else n for i, n in enumerate(want_lens)]
