"""Bounds of attention behind shared prefixes on the GPU: a request is read up to its prefix and max_suffix_len keys, no further."""
import pytest
import torch

from helpers import announce
from shared_helpers import Case
from test_shared_bounds_cpu import check_refused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("prefix", [448, 500, 511])
@pytest.mark.parametrize("nq,causal", [(1, False), (3, True)])
def test_keys_past_max_suffix_len_are_not_read(fp8, d, prefix, nq, causal):
    """The longest request has 1 to 130 keys more than the bound allows; the exact result is that of requests cut there."""
    announce(f"shared bounds fp8={fp8} d={d} prefix={prefix} nq={nq}")
    own = [0, 1, 40, 100, 101, 130, 163, 164, 230, -200, -prefix]
    case = Case([len(own)], [prefix], [prefix + x for x in own], d=d, page=64, fp8=fp8)
    q = case.q(8, nq)
    full = case.lens
    for bound in (0, 1, 37, 64, 100, 229):
        case.lens = [min(n, prefix + bound) for n in full]
        o, lse = case.call(q, causal=causal, return_lse=True, max_prefix_len=prefix, max_suffix_len=bound)
        case.check(o, q, causal, lse)
        assert torch.equal(case.call(q, causal=causal, max_prefix_len=prefix, max_suffix_len=bound), o)


def test_the_bound_is_counted_from_the_prefix_as_it_is_shared():
    """Groups with prefixes of their own, some above max_prefix_len."""
    groups, prefixes = [3, 2, 4, 1], [300, 70, 0, 129]
    own = [0, 50, 51, 10, 90, 1, 49, 50, 130, 64]
    start = [p for p, n in zip(prefixes, groups) for _ in range(n)]
    full = [p + x for p, x in zip(start, own)]
    case = Case(groups, prefixes, full, d=128, page=16)
    q = case.q(8, 1)
    for most in (0, 60, 128, 131, 300, 1000):
        for bound in (0, 50, 64):
            case.lens = [min(n, min(p, most) + bound) for n, p in zip(full, start)]
            case.check(case.call(q, causal=True, max_prefix_len=most, max_suffix_len=bound), q, True)


def test_bounds_that_do_not_fit_are_refused():
    case = Case([3, 2], [70, 20], [75, 70, 130, 21, 90], page=16)
    case.call(case.q(4, 2))
    check_refused(case, case.q(4, 2))
