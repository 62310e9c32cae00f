"""Attention behind shared prefixes and pages: what a padded batch, other streams, other host paths and large pools bring."""
import math

import pytest
import torch

import fused_attn
from fused_attn import _hip
from pages_helpers import append_oracle, check_allocate, check_release, ALLOCATE, RELEASE
from shared_helpers import Case, check_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 99, 40], [130, 17, 0, 200, 255], [0, 0, 256, 1, 700]])
def test_groups_whose_requests_are_shorter_than_the_prefix(fp8, d, lens):
    """Nobody holds the whole prefix: keys are read only as far as the longest request has them (what lies behind it in the
    pages, and in the table, is NaN and garbage), and partitions behind that are empty."""
    case = Case([len(lens)], [700], lens, d=d, page=64, fp8=fp8)
    for nq, split in ((1, None), (3, 64), (9, 256)):
        q = case.q(8, nq)
        o, lse = case.call(q, causal=True, return_lse=True, split_len=split, max_prefix_len=700, max_suffix_len=10)
        case.check(o, q, True, lse)


def test_nan_and_infinity_in_keys_that_a_request_does_not_see():
    """V of a later partition is NaN: the requests that see it are NaN, a shorter one is not, nor one that ends before it."""
    case = Case([4], [640], [650, 100, 0, 700], d=128, page=64)
    q = case.q(8, 2)
    want = case.call(q, causal=True, split_len=64)
    page = int(case.table[0, 400 // 64])
    case.v[page, :, 400 % 64] = math.nan
    got = case.call(q, causal=True, split_len=64)
    assert torch.isnan(got[0]).all() and torch.isnan(got[3]).all()
    assert torch.equal(got[1:3], want[1:3])
    case.v[page, :, 400 % 64] = math.inf
    got = case.call(q, causal=True, split_len=64)
    assert torch.isposinf(got[0]).all() and torch.equal(got[1:3], want[1:3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shared", [True, False])
def test_every_fp8_value_is_widened_exactly(dtype, shared):
    """64 keys with the same scores and the same V row: the output is that row's value, all 254 finite codes, bit for bit
    (sums of 64 equal numbers and the division by 64 are exact; the scale is a power of two)."""
    codes = torch.tensor([c for c in range(256) if c & 127 != 127] + [0, 0], dtype=torch.uint8, device="cuda")
    v = codes.expand(2, 1, 64, 256).contiguous().view(torch.float8_e4m3fn)
    k = torch.zeros_like(v.view(torch.uint8)).view(torch.float8_e4m3fn)
    scale = torch.full((2, 1, 1), 0.25, device="cuda")
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.full((2,), 64, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 2, 1, 256, device="cuda").to(dtype)
    o = fused_attn.attention_shared_prefix(q, k, v, table, lens, 64 if shared else 0, k_scale=scale, v_scale=scale)
    assert torch.equal(o, (codes.view(torch.float8_e4m3fn).float() * 0.25).to(dtype).expand_as(o))


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127])
@pytest.mark.parametrize("fp8", [False, True])
def test_short_prefixes(prefix, fp8):
    case = Case([5], [prefix], [prefix + x for x in (1, 2, 63, 64, 130)], d=64, page=64, fp8=fp8)
    q = case.q(4, 1)
    case.check(case.call(q, causal=True), q, True)


@pytest.mark.parametrize("page", [16, 112, 1024, 4096])
def test_page_sizes_and_many_queries(page):
    """Pages far smaller and larger than a partition; more rows a request than a wave or a workgroup has."""
    case = Case([3], [2100], [2100, 2700, 5200], hkv=1, d=128, page=page)
    for hq, nq in ((1, 1), (4, 70), (3, 33)):
        q = case.q(hq, nq)
        case.check(case.call(q, causal=True), q, True)


def test_pages_outside_the_pool_read_as_zero_keys():
    case = Case([3], [256], [300, 256, 290], d=64, page=16, dtype=torch.float16)
    case.table[:, 3] = 10 ** 6  # in the prefix
    case.table[0, 17] = -5  # a request's own
    for x in case.kv:
        x[:, :, 48:64] = 0
        x[0, :, 272:288] = 0
    q = case.q(4, 2)
    case.check(case.call(q, causal=True), q, True)


@pytest.mark.parametrize("fp8", [False, True])
def test_the_python_path_gives_the_same_bits(fp8, monkeypatch):
    case = Case([6, 3], [320, 200], [330, 0, 500, 321, 320, 400, 210, 222, 300], d=128, page=64, fp8=fp8)
    q = case.q(8, 2)
    bounds = {"max_prefix_len": 320, "max_suffix_len": 180}
    want = case.call(q, causal=True, **bounds)  # (enables the device)
    case.check(want, q, True)
    assert _hip.native is not None, "the native host path is not built"
    got = _hip.native.shared_prefix(q, case.k, case.v, case.table, case.seqlens, case.prefix_lens, case.cu_groups,
                                    case.scales.get("k_scale"), case.scales.get("v_scale"), 320, 180, True, q.shape[-1] ** -0.5, 0)
    assert torch.equal(got, want)
    # what needs preparation, or is refused, is left to Python
    n = _hip.native
    more = (case.scales.get("k_scale"), case.scales.get("v_scale"), 320, 180, True, 0.1, 0)
    for args in ((q.float(), case.k), (q[..., ::2], case.k), (q, case.k.cpu()), (q, case.k[..., :64]), (q[:0], case.k)):
        assert n.shared_prefix(*args, case.v, case.table, case.seqlens, case.prefix_lens, case.cu_groups, *more) is None
    assert n.shared_prefix(q, case.k, case.v, case.table.long(), case.seqlens, case.prefix_lens, case.cu_groups, *more) is None
    assert n.shared_prefix(q, case.k, case.v, case.table, case.seqlens, None, 5, *more) is None
    monkeypatch.setattr(_hip, "native", None)
    assert torch.equal(case.call(q, causal=True, **bounds), want)
    wide = torch.stack([q, q], -1)[..., 0]  # a view that is copied first
    assert torch.equal(case.call(wide, causal=True, **bounds), want)


def test_pages_through_python(monkeypatch):
    check_allocate(ALLOCATE[4], "cuda")
    assert _hip.native is not None
    monkeypatch.setattr(_hip, "native", None)
    for case in ALLOCATE[2:7]:
        check_allocate(case, "cuda", wide=1)
    for case in RELEASE[2:5]:
        check_release(case, "cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    pools = [torch.randn(9, 2, 16, 64, device="cuda", generator=g).half() for _ in "kv"]
    k, slots = torch.randn(40, 2, 64, device="cuda", generator=g).half(), torch.randperm(144, device="cuda", generator=g)[:40]
    want = append_oracle(k, -k, *pools, slots)
    fused_attn.append_kv_paged(k, -k, *pools, slots)
    assert all(torch.equal(p.cpu(), w) for p, w in zip(pools, want))


def test_forced_reference_backend(monkeypatch):
    case = Case([3], [128], [130, 200, 129], d=64, page=16)
    q = case.q(4, 1)
    case.call(q, max_prefix_len=128, max_suffix_len=80)
    monkeypatch.setenv("FUSED_ATTN_BACKEND", "reference")
    case.check(case.call(q, max_prefix_len=128, max_suffix_len=80), q)
    check_allocate(ALLOCATE[4], "cuda")
    check_release(RELEASE[2], "cuda")


def test_two_streams_at_once():
    """Calls on two streams share nothing: each equals the call made alone."""
    cases = [Case([20], [1000], [1000 + 13 * i for i in range(20)], d=128, page=16, seed=s) for s in (1, 2)]
    qs = [c.q(8, 1, seed=s) for s, c in enumerate(cases)]
    want = [c.call(q, max_suffix_len=260) for c, q in zip(cases, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(cases[i].call(qs[i], max_suffix_len=260))
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        assert all(torch.equal(o, w) for o in got)


def test_two_captured_graphs_in_turn():
    cases = [Case([6], [512], [512 + 60 * i for i in range(6)], d=64, page=32, seed=s) for s in (3, 4)]
    qs = [c.q(8, 1, seed=s) for s, c in enumerate(cases)]
    kw = {"max_prefix_len": 512, "max_suffix_len": 300, "causal": True}
    graphs, outs = [], []
    for c, q in zip(cases, qs):
        c.call(q, **kw)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c.call(q, **kw))
    for _ in range(3):
        for q in qs:
            q.copy_(torch.randn_like(q))
        for g in graphs:
            g.replay()
        for c, q, o in zip(cases, qs, outs):
            assert torch.equal(o, c.call(q, **kw))


@pytest.mark.parametrize("fp8", [False, True])
def test_pools_behind_4_gib(fp8):
    """Rows past 2^31 elements of the pools."""
    small = Case([4], [256], [300, 256, 420, 0], hkv=2, d=128, page=64, fp8=fp8)
    q = small.q(8, 1)
    want = small.call(q, causal=True)
    count = small.k.shape[0]
    pages = 2 ** 31 // (2 * 64 * 128) + count
    big = []
    for pool in (small.k, small.v):
        t = torch.empty(pages, *pool.shape[1:], dtype=pool.dtype, device="cuda")
        t.view(torch.uint8).zero_()
        t[-count:] = pool
        big.append(t)
    scales = {}
    for name, s in small.scales.items():
        scales[name] = torch.zeros(pages, *s.shape[1:], device="cuda")
        scales[name][-count:] = s
    table = torch.where((small.table >= 0) & (small.table < count), small.table + pages - count, small.table)
    got = fused_attn.attention_shared_prefix(q, *big, table, small.seqlens, 256, causal=True, **scales)
    assert torch.equal(got, want)
    check_rows(got[:3], q[:3], *[x[:3] for x in small.kv], causal=True, lens=small.lens[:3])
    del big


@pytest.mark.parametrize("number", [False, True])
def test_a_bound_below_the_prefix_alone(number):
    """max_prefix_len below the prefix, max_suffix_len left to be read: the rest of the prefix counts as own keys."""
    case = Case([5], [500], [510, 600, 500, 507, 800], d=128, page=16)
    q = case.q(8, 2)
    kw = {"prefix_lens": 500} if number else {}
    for bound in (0, 100, 192, 499):
        case.check(case.call(q, causal=True, max_prefix_len=bound, **kw), q, True)
