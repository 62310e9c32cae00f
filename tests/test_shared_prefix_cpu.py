"""Attention behind shared prefixes on the CPU: the torch form, refusals, and the C ABI's checks of arguments."""
import ctypes

import pytest
import torch

import fused_attn
from fused_attn import _hip, shared_prefix
from shared_helpers import Case


@pytest.mark.parametrize("fp8", [False, True])
def test_torch_form(fp8):
    """(Scales of CPU tensors come from a true division: the values are what the pools' own scales give.)"""
    case = Case([3, 2], [70, 20], [75, 70, 100, 21, 64], page=64 if fp8 else 16, device="cpu", fp8=fp8)
    q = case.q(4, 2, torch.float16 if not fp8 else torch.bfloat16)
    if not fp8:
        case.k, case.v = case.k.half(), case.v.half()
    o, lse = case.call(q, causal=True, return_lse=True)
    assert o.shape == q.shape and lse.shape == q.shape[:3]
    for i, n in enumerate(case.lens):
        k, v = (x[i:i + 1, :, :n].float() for x in case.kv)
        want = fused_attn.attention_reference(q[i:i + 1].float(), k, v, causal=True)
        assert (o[i:i + 1].float() - want).abs().max() <= 2.0 ** -6 * want.abs().max()


def _args(case, **kw):
    a = {"q": case.q(4, 1), "k_cache": case.k, "v_cache": case.v, "block_table": case.table, "seqlens_k": case.seqlens,
         "prefix_lens": case.prefix_lens, "cu_groups": case.cu_groups}
    a.update(kw)
    return a


def test_refusals():
    case = Case([3, 2], [70, 20], [75, 70, 100, 21, 64], device="cpu")
    fused_attn.attention_shared_prefix(**_args(case))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    q = case.q(4, 1)
    for kw in ({"q": q.float()}, {"q": q[0]}, {"q": q.half()}, {"q": q[..., :32]}, {"q": q[:, :3]}, {"q": q[:4]},
               {"k_cache": case.k[:1]}, {"k_cache": case.k.view(torch.uint8), "v_cache": case.v.view(torch.uint8)},
               {"block_table": case.table.long()}, {"block_table": case.table[0]}, {"seqlens_k": case.seqlens.long()},
               {"seqlens_k": case.seqlens[:4]}, {"prefix_lens": i32(70)}, {"prefix_lens": torch.tensor([70, 20])},
               {"prefix_lens": i32(70, 20), "cu_groups": None}, {"cu_groups": i32(0)}, {"cu_groups": torch.tensor([0, 3, 5])},
               {"cu_groups": i32(0, 1, 2, 3, 4, 5, 5), "prefix_lens": 64}):
        with pytest.raises(RuntimeError):
            fused_attn.attention_shared_prefix(**_args(case, **kw))


def test_abi():
    assert ctypes.sizeof(_hip.SharedPrefix) == 2 * 8 + 4 * 4
    lib = _hip.load_library()
    p = _hip.FwdParams(16, 16, 16, 16, 4 * 128, 128, 128, 0, 64, 128, 0, 64, 128, 4 * 128, 128, 128, 5, 4, 2, 1, 0, 128, 0.1, 0,
                       _hip.BF16, _hip.BF16)
    kv = _hip.PagedKV(16, 4, 4, 64, 16, 9, 0, 8192, 8192)
    s = _hip.SharedPrefix(16, 16, 2, 100, 50, 128)
    need = lib.fa_shared_prefix_workspace_bytes(p, kv, s)
    # one partition of the prefix and one of the own keys: partials, maxima and sums of 20 rows
    assert need == 20 * 2 * (128 + 2) * 4
    assert lib.fa_shared_prefix_workspace_bytes(p, kv, _hip.SharedPrefix(16, 16, 2, 100, 50, 0)) >= need

    def status(ws=16, nbytes=need, **kw):
        ps = [type(x).from_buffer_copy(x) for x in (p, kv, s)]
        for name, value in kw.items():
            owner = next(x for x in ps if any(f[0] == name for f in x._fields_))
            setattr(owner, name, value)
        got = lib.fa_attention_shared_prefix(*ps, ctypes.c_void_p(ws), nbytes, ctypes.c_void_p(0))
        assert got == _hip.FA_OK or lib.fa_last_error()
        if got not in (_hip.FA_OK, _hip.FA_ERR_WORKSPACE):
            assert lib.fa_shared_prefix_workspace_bytes(*ps) == 0
        return got

    for kw in ({"max_prefix_len": -1}, {"max_suffix_len": -1}, {"num_groups": -1}, {"num_groups": 0}, {"num_groups": 6},
               {"cu_groups": None}, {"cu_groups": 18}, {"prefix_lens": 18}, {"split_len": 32}, {"split_len": -64},
               {"page_size": 24}, {"block_table": None}, {"seqlens_k": None}, {"block_table_stride": 3}, {"heads_kv": 3},
               {"k_page_stride": 4}, {"scale": float("nan")}, {"k": None}, {"q": 8}, {"kv_dtype": _hip.FP8_E4M3}):
        assert status(**kw) == _hip.FA_ERR_INVALID_ARGUMENT, kw
    for kw in ({"max_prefix_len": (1 << 29) + 1}, {"max_suffix_len": (1 << 29) + 1}, {"head_dim": 32}, {"dtype": _hip.F32},
               {"split_len": 1 << 20, "page_size": 16}, {"batch": 1 << 30}):
        assert status(**kw) in (_hip.FA_ERR_UNSUPPORTED, _hip.FA_ERR_INVALID_ARGUMENT), kw
    assert status(nbytes=need - 1) == _hip.FA_ERR_WORKSPACE
    assert status(ws=0) == _hip.FA_ERR_WORKSPACE
    assert status(ws=8) == _hip.FA_ERR_WORKSPACE
    assert status(batch=0) == _hip.FA_OK and status(seqlen_q=0) == _hip.FA_OK


@pytest.mark.parametrize("bound,longest", [(1000, 60), (100, 60), (64, 96), (0, 160)])
def test_own_keys_are_counted_from_the_shared_ones(bound, longest):
    # a prefix longer than max_prefix_len is shared up to it, and the rest of it is each request's own
    lens, cu = torch.tensor([160, 90, 0, 70], dtype=torch.int32), torch.tensor([0, 3, 4], dtype=torch.int32)
    prefixes = torch.tensor([100, 50], dtype=torch.int32)
    assert shared_prefix._longest_suffix(lens, prefixes, cu, bound) == longest
    assert shared_prefix._longest_suffix(lens[:3], 100, None, bound) == longest
