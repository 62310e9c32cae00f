"""Libraries of the same ABI version that lack functions added within it."""
import ctypes

import pytest
import torch

import fused_attn
from fused_attn import _hip

PAGES = ["fa_allocate_pages", "fa_release_pages", "fa_append_kv_paged", "fa_shared_prefix_workspace_bytes",
         "fa_attention_shared_prefix"]


class Older:
    """The built library without one of its functions."""

    def __init__(self, missing):
        lib = ctypes.CDLL(_hip.library_path())
        self._FuncPtr, self._lib, self._missing = lib._FuncPtr, lib, missing

    def __getattr__(self, name):
        if name == self._missing:
            raise AttributeError(name)
        return getattr(self._lib, name)


@pytest.mark.parametrize("missing", PAGES)
def test_a_library_without_one_of_the_functions_of_pages(missing, monkeypatch):
    """It loads, and only the calls that need them are refused."""
    lib = Older(missing)
    _hip._bind(lib)
    assert not _hip._has_pages(lib)
    monkeypatch.setattr(_hip, "_lib", lib)
    with pytest.raises(RuntimeError, match="build it again"):
        _hip._pages_library()
    q = torch.randn(1, 2, 4, 16)
    assert fused_attn.attention(q, q, q).shape == q.shape


def test_the_built_library_has_them():
    lib = Older(None)
    _hip._bind(lib)
    assert _hip._has_pages(lib)
