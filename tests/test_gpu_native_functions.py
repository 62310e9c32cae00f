"""The native host functions of pages and shared prefixes beside other threads of Python."""
import ctypes

import pytest
import torch

from fused_attn import _hip
from shared_helpers import Case

pytestmark = pytest.mark.gpu


def _pointer(f):
    return ctypes.cast(f, ctypes.c_void_p)


@pytest.fixture
def held():
    """The library's calls replaced by one that returns whether the calling thread holds the GIL: 0, success, if not."""
    case = Case([3], [128], [130, 200, 129], d=64, page=16)
    case.call(case.q(4, 1), max_prefix_len=128, max_suffix_len=80)  # (enables the device)
    assert _hip.native is not None, "the native host path is not built"
    lib, check = _hip.load_library(), _pointer(ctypes.pythonapi.PyGILState_Check)
    _hip._native.fa_torch_bind_pages(check, check, check)
    _hip._native.fa_torch_bind_shared(_pointer(lib.fa_shared_prefix_workspace_bytes), check)
    try:
        yield case
    finally:
        _hip._native.fa_torch_bind_pages(*map(_pointer, (lib.fa_allocate_pages, lib.fa_release_pages, lib.fa_append_kv_paged)))
        _hip._native.fa_torch_bind_shared(*map(_pointer, (lib.fa_shared_prefix_workspace_bytes, lib.fa_attention_shared_prefix)))


def test_calls_are_made_without_the_gil(held):
    n, i = _hip.native, torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ctypes.pythonapi.PyGILState_Check() == 1
    assert n.allocate_pages(held.table, held.seqlens, i, i, i[:1], 16, 5) is not None
    assert n.release_pages(held.table, held.seqlens, i.bool(), i, i[:1], None, 16) is not None
    row = held.k[:, :, 0]
    assert n.append_kv_paged(row, row, held.k, held.v, torch.zeros(row.shape[0], dtype=torch.int64, device="cuda")) is True
    q = held.q(4, 1)
    assert n.shared_prefix(q, held.k, held.v, held.table, held.seqlens, None, None, None, None, 128, 80, False, 0.1, 0) is not None


def test_an_allocation_that_fails_is_reported():
    """What is thrown without the GIL is caught with it: a workspace of 500 GB, more than the card has."""
    case = Case([64], [64], [65] * 64, hkv=1, d=64, page=16)
    q = case.q(32, 1)
    want = case.call(q, max_suffix_len=1)
    with pytest.raises(torch.OutOfMemoryError):
        case.call(q, prefix_lens=64, max_suffix_len=1 << 29)
    assert torch.equal(case.call(q, max_suffix_len=1), want)
