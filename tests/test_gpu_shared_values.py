"""Attention behind shared prefixes over values that a quantiser or a healthy model does not write: FP8 scales that are 0,
negative, far apart, infinite or NaN, and rows of V that are no numbers."""
import math

import pytest
import torch

from cache_norms import row_errors
from helpers import announce
from shared_helpers import Case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
PREFIX = 460  # 448 of its keys are read for the group, 7 blocks
LENS = [PREFIX + x for x in (0, 1, 300, 63, 64, 65, -300, -460, 129, 200, -360, -330, 5)]


def scale_blocks(case, factors):
    """Multiply the V scale of key block j by factors[j % len], 64 keys a block and a page, and bring the values in line."""
    assert case.k.shape[2] == 64
    seen = {}
    for row, n in zip(case.table.tolist(), case.lens):
        for j, page in enumerate(row[:-(-n // 64)]):
            assert seen.setdefault(page, j) == j
    scale = case.scales["v_scale"]
    for page, j in seen.items():
        scale[page] = scale[page] * factors[j % len(factors)] if math.isfinite(factors[j % len(factors)]) else factors[j % len(factors)]
    for i, n in enumerate(case.lens):
        pages = case.table[i, :-(-n // 64)].long()
        codes = case.v.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
        rows = (codes * scale[pages].double()[..., None]).transpose(0, 1).flatten(1, 2)
        case.kv[1][i, :, :n] = rows[:, :n]


FACTORS = [
    (1, 0, 1, 0, 0),  # codes that are not 0 behind and ahead of blocks with a scale
    (0, 0, 0, 1, 1, 0),
    (0,),
    (1e-3, 1, 1e3, 0.05, 30),  # six decades: O changes its unit with every block
    (1, 2.1, 4.5, 2, 0.9, 0.4),  # about a factor 2 from block to block: inside the exponents or not
    (1, -1, -1.5, 2, 0, -0.1),
    # what a writer's smallest scale may be: O in such a unit would overflow.  Blocks below 2^-90 of another's scale count as
    # 0; their values, at most 448e-36, are below every tolerance here
    (1, 1e-36, 1, 2e-41, 1),
]


@pytest.mark.parametrize("dtype,factors", [(t, f) for t in DTYPES for f in FACTORS] + [(torch.bfloat16, (1e-25, 1e-33, 3e-26))],
                         ids=str)  # (the last one's outputs are below fp16's range)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp8_block_scales(dtype, d, factors):
    announce(f"shared fp8 scales {dtype} d={d} {factors}")
    case = Case([len(LENS)], [PREFIX], LENS, d=d, page=64, fp8=True)
    scale_blocks(case, factors)
    for nq, split in ((1, None), (3, 192)):
        q = case.q(8, nq, dtype)
        o, lse = case.call(q, causal=True, return_lse=True, split_len=split)
        case.check(o, q, True, lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("block", [2, 9])  # among the shared keys, among a request's own
def test_fp8_scales_without_a_value(d, bad, block):
    """The rows that see the block are NaN, their log-sum-exps and all other rows what they are without it."""
    announce(f"shared fp8 scale {bad} d={d} block={block}")
    case = Case([len(LENS)], [PREFIX], LENS, d=d, page=64, fp8=True)
    factors = [1.0] * 13
    q, nq = case.q(8, 3), 3
    _, want_lse = case.call(q, causal=True, return_lse=True)
    kv = case.kv[1].clone()
    factors[block] = bad
    scale_blocks(case, factors)
    case.kv[1] = kv
    got, lse = case.call(q, causal=True, return_lse=True)
    assert torch.equal(lse, want_lse)
    sees = torch.tensor([[n - nq + i >= 64 * block for i in range(nq)] for n in LENS], device="cuda")[:, None].expand(-1, 8, -1)
    assert sees.any() and not sees.all()
    assert torch.isnan(got[sees]).all()
    err, tol = row_errors(got.masked_fill(sees[..., None], 0), q, *case.kv, causal=True, lens=LENS)
    assert (err <= tol)[~sees].all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("split", [None, 192])
def test_rows_of_v_that_a_shorter_request_does_not_hold(fp8, dtype, d, split):
    """V rows of shared keys are NaN or infinite: the rows that see one are no numbers, all others are what they are without
    them, also where the bad row lies in their own last tile, page or partition."""
    announce(f"shared bad rows of V fp8={fp8} {dtype} d={d} split={split}")
    lens = [650, 100, 0, 700, 391, 399, 400, 401, 402, 640, 384, 130, 131]
    case = Case([len(lens)], [640], lens, d=d, page=64, fp8=fp8, dtype=dtype)
    for bad, key in ((math.nan, 400), (math.inf, 400), (-math.inf, 129), (math.nan, 639)):
        if fp8 and bad != math.nan:
            bad = math.nan
        page = int(case.table[0, key // 64])
        row = case.v[page, :, key % 64]
        keep = row.view(torch.uint8).clone()
        if fp8:
            row.view(torch.uint8).fill_(0x7f)
        else:
            row.fill_(bad)
        for nq, causal in ((1, False), (3, True), (40, True)):
            q = case.q(8, nq, dtype)
            got = case.call(q, causal=causal, split_len=split)
            sees = torch.tensor([[key < (n - nq + 1 + i if causal else n) for i in range(nq)] for n in lens], device="cuda")
            sees = sees[:, None].expand(-1, 8, -1)
            assert sees.any() and not sees.all()
            if math.isnan(bad):
                assert torch.isnan(got[sees]).all()
            else:
                assert (got[sees] == bad).all()
            err, tol = row_errors(got.masked_fill(sees[..., None], 0), q, *case.kv, causal=causal, lens=lens)
            assert (err <= tol)[~sees].all(), (bad, key, nq)
        row.view(torch.uint8).copy_(keep)


@pytest.mark.parametrize("page", [16, 64])
def test_bad_rows_of_v_in_groups_of_their_own(page):
    """Several groups, long partitions, a negative scale, pools in another layout: the short requests' rows are those of the same
    pools without the bad rows."""
    lens = [3300, 40, 700, 3001, 900, 20, 1000]
    case = Case([4, 3], [3000, 900], lens, hkv=2, d=128, page=page)
    pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in (case.k, case.v)]
    case.k, case.v = pools
    q = case.q(8, 2)
    want = case.call(q, causal=True, scale=-0.1)
    for i, key in ((0, 1500), (4, 60)):
        case.v[int(case.table[i, key // page]), :, key % page] = math.inf
    got = case.call(q, causal=True, scale=-0.1)
    for i in (1, 2, 5):  # 40, 700, 20 keys
        assert ((got[i].double() - want[i].double()).norm(dim=-1) <= 2.0 ** -6 * (1 + want[i].double().norm(dim=-1))).all()
    for i in (0, 3, 4, 6):
        assert torch.isposinf(got[i]).all()
