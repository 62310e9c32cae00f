"""Bounds of attention behind shared prefixes in the torch form."""
import pytest
import torch

import fused_attn
from fused_attn import shared_prefix
from shared_helpers import Case


@pytest.mark.parametrize("most", [None, 0, 30, 70, 500])
@pytest.mark.parametrize("bound", [0, 1, 40])
def test_the_torch_form_keeps_the_bounds(most, bound):
    prefixes = [70, 20]
    case = Case([3, 2], prefixes, [75, 70, 130, 21, 90], page=16, device="cpu")
    q = case.q(4, 2, torch.bfloat16)
    got = case.call(q, causal=True, max_prefix_len=most, max_suffix_len=bound)
    cut = [min(n, min(p, 500 if most is None else most) + bound) for n, p in zip(case.lens, [70, 70, 70, 20, 20])]
    want = fused_attn.attention_paged(q, case.k, case.v, case.table, torch.tensor(cut, dtype=torch.int32), causal=True)
    assert torch.equal(got, want)
    assert case.seqlens.tolist() == case.lens


def test_prefixes_of_requests():
    """A number for every group, requests of no group, prefixes below 0."""
    lens = torch.zeros(6, dtype=torch.int32)
    cu = torch.tensor([1, 3, 3, 5], dtype=torch.int32)
    assert shared_prefix._prefixes(lens, 40, cu, None).tolist() == [0, 40, 40, 40, 40, 0]
    assert shared_prefix._prefixes(lens, 40, None, 30).tolist() == [30] * 6
    p = torch.tensor([5, 6, -7], dtype=torch.int32)
    assert shared_prefix._prefixes(lens, p, cu, 4).tolist() == [0, 4, 4, 0, 0, 0]
    assert shared_prefix._prefixes(lens, p[:1], None, None).tolist() == [5] * 6


BEYOND = [2 ** 29 + 1, 2 ** 31, 2 ** 32, 2 ** 32 + 64]  # the last two are 0 and 64 in 32 bits


def check_refused(case, q):
    for n in BEYOND:
        for kw in ({"max_prefix_len": n}, {"max_suffix_len": n}, {"max_suffix_len": n, "max_prefix_len": 70}, {"split_len": n},
                   {"prefix_lens": n}, {"prefix_lens": n, "max_suffix_len": 60}, {"prefix_lens": 70, "max_suffix_len": n}):
            with pytest.raises(RuntimeError, match="2\\^29"):
                case.call(q, **kw)
    # the lesser of two bounds of the prefix counts
    assert torch.equal(case.call(q, prefix_lens=2 ** 32, max_prefix_len=64, max_suffix_len=600),
                       case.call(q, prefix_lens=64, max_suffix_len=600))


def test_bounds_that_do_not_fit_are_refused():
    case = Case([3, 2], [70, 20], [75, 70, 130, 21, 90], page=16, device="cpu")
    check_refused(case, case.q(4, 2, torch.bfloat16))
