"""Pages on the CPU: the torch forms against the oracle, refusals, and the C ABI's checks of arguments."""
import ctypes

import pytest
import torch

import fused_attn
from fused_attn import _hip
from oracle import pages_oracle
from pages_helpers import ALLOCATE, RELEASE, append_oracle, check_allocate, check_release


@pytest.mark.parametrize("case", ALLOCATE, ids=str)
def test_allocate(case):
    check_allocate(case, "cpu", wide=3)


@pytest.mark.parametrize("case", RELEASE, ids=str)
def test_release(case):
    check_release(case, "cpu")


def test_oracle_by_hand():
    """Two requests, pages of 4: 3 + 2 keys need one more page, 4 + 5 need two; the list is taken from its end."""
    table, slots, cu, lens, left = pages_oracle.allocate([[7, 0, 0], [9, 0, 0]], [3, 4], [2, 5], [1, 2, 3, 4], 4, 4, 7)
    assert table == [[7, 4, 0], [9, 3, 2]] and left == 1 and lens == [5, 9] and cu == [0, 2, 7]
    assert slots == [7 * 4 + 3, 4 * 4, 3 * 4, 3 * 4 + 1, 3 * 4 + 2, 3 * 4 + 3, 2 * 4]
    # one page short: the second request keeps its length, the first has its page
    table, slots, cu, lens, left = pages_oracle.allocate([[7, 0, 0], [9, 0, 0]], [3, 4], [2, 5], [1, 2], 2, 4, 7)
    assert table == [[7, 2, 0], [9, 0, 0]] and left == 1 and lens == [5, 4] and slots[2:] == [-1] * 5
    # 9 keys are three pages, of which 5 shared ones fill one
    assert pages_oracle.release([[7, 4, 5]], [9], [True], [1, 0, 0], 1, 4, [5]) == ([1, 4, 5], [0], 3)


def test_a_request_without_need_of_pages_goes_on_when_the_list_is_empty():
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32)
    lens, new = torch.tensor([16, 3, 5], dtype=torch.int32), torch.tensor([1, 1, 1], dtype=torch.int32)
    slots, _, seqlens, _ = fused_attn.allocate_pages(table, lens, new, torch.zeros(1, dtype=torch.int32),
                                                     torch.zeros(1, dtype=torch.int32), 16, 3)
    assert slots.tolist() == [-1, 16 + 3, 32 + 5] and seqlens.tolist() == [16, 4, 6]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append(dtype):
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(9, 3, 24, generator=g).to(dtype) for _ in "kv")
    k_cache, v_cache = (torch.randn(4, 3, 5, 24, generator=g).to(dtype) for _ in "kv")
    slots = torch.tensor([3, 19, -1, 20, 0, 7, 8, 2 ** 40, 11])
    want = append_oracle(k, v, k_cache, v_cache, slots)
    fused_attn.append_kv_paged(k, v, k_cache, v_cache, slots)
    assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])


def _allocate_args(**kw):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    a = {"block_table": i(2, 3), "seqlens_k": i(2), "new_lens": i(2), "free_pages": i(4), "num_free": i(1), "page_size": 16,
         "num_tokens": 5}
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    {"block_table": torch.zeros(2, 3)}, {"block_table": torch.zeros(2, dtype=torch.int32)},
    {"seqlens_k": torch.zeros(3, dtype=torch.int32)}, {"seqlens_k": torch.zeros(2, dtype=torch.int64)},
    {"new_lens": torch.zeros(1, dtype=torch.int32)}, {"free_pages": torch.zeros(2, 2, dtype=torch.int32)},
    {"free_pages": torch.zeros(8, dtype=torch.int32)[::2]}, {"num_free": torch.zeros(2, dtype=torch.int32)},
    {"num_free": torch.zeros(1)}, {"page_size": 0}, {"page_size": 1 << 25}, {"num_tokens": -1}, {"num_tokens": 2 ** 31 - 1}],
    ids=lambda kw: next(iter(kw)))
def test_allocate_refuses(kw):
    with pytest.raises(RuntimeError):
        fused_attn.allocate_pages(**_allocate_args(**kw))


def test_release_refuses():
    a = _allocate_args()
    a.pop("new_lens"), a.pop("num_tokens")
    for kw in ({"done": torch.zeros(2)}, {"done": torch.zeros(3, dtype=torch.bool)},
               {"done": torch.zeros(2, dtype=torch.bool), "keep_lens": torch.zeros(2)}):
        with pytest.raises(RuntimeError):
            fused_attn.release_pages(**a, **kw)


def test_append_refuses():
    def call(t=2, h=2, d=16, dtype=torch.float16, pool=None, slots=None, v=None):
        k = torch.zeros(t, h, d, dtype=dtype)
        pool = torch.zeros(3, 2, 4, 16, dtype=torch.float16) if pool is None else pool
        fused_attn.append_kv_paged(k, k if v is None else v, pool, pool.clone(),
                                   torch.zeros(t, dtype=torch.int64) - 1 if slots is None else slots)

    call()
    pool = torch.zeros(3, 2, 4, 32, dtype=torch.float16)
    for kw in ({"dtype": torch.float32}, {"dtype": torch.bfloat16}, {"h": 1}, {"d": 8}, {"slots": torch.zeros(3, dtype=torch.int64)},
               {"slots": torch.zeros(2, dtype=torch.int32)}, {"pool": pool[..., ::2]}, {"pool": pool[..., 4:20]},
               {"v": torch.zeros(3, 2, 16, dtype=torch.float16)},
               {"d": 12, "pool": torch.zeros(3, 2, 4, 12, dtype=torch.float16)},
               {"pool": torch.zeros(1, 2, 4, 16, dtype=torch.float16).expand(3, 2, 4, 16)}):
        with pytest.raises(RuntimeError):
            call(**kw)


def test_abi():
    assert ctypes.sizeof(_hip.PagesParams) == 2 * 8 + 6 * 4 + 10 * 8
    assert ctypes.sizeof(_hip.AppendPagedParams) == 6 * 8 + 8 * 8 + 8 + 6 * 4
    lib = _hip.load_library()
    x = ctypes.c_void_p(0)
    p = _hip.PagesParams(16, 3, 2, 3, 16, 4, 5, 0, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16)

    def refused(f, base, **kw):
        q = type(base).from_buffer_copy(base)
        for name, value in kw.items():
            setattr(q, name, value)
        status = f(q, x)
        assert status in (_hip.FA_ERR_INVALID_ARGUMENT, _hip.FA_ERR_UNSUPPORTED) and lib.fa_last_error(), kw

    for f in (lib.fa_allocate_pages, lib.fa_release_pages):
        assert f(None, x) == _hip.FA_ERR_INVALID_ARGUMENT
        for kw in ({"batch": -1}, {"block_table_cols": -1}, {"free_capacity": -1}, {"free_capacity": 2 ** 31 - 1},
                   {"page_size": 0}, {"page_size": (1 << 24) + 1}, {"batch": (1 << 24) + 1}, {"block_table_stride": 2},
                   {"seqlens": None}, {"seqlens_out": None}, {"block_table": None}, {"num_free": None}, {"num_free_out": None},
                   {"free_pages": None}, {"block_table": 18}, {"free_pages": 18}):
            refused(f, p, **kw)
    for kw in ({"num_tokens": -1}, {"num_tokens": 2 ** 31 - 1}, {"new_lens": None}, {"cu_seqlens": None}, {"slots": None},
               {"slots": 20}):
        refused(lib.fa_allocate_pages, p, **kw)
    refused(lib.fa_release_pages, p, done=None)

    a = _hip.AppendPagedParams(16, 16, 32, 16, 32, 16, 16, 16, 128, 64, 16, 128, 64, 16, 16, 4, 2, 16, 3, 4)
    assert lib.fa_append_kv_paged(None, x) == _hip.FA_ERR_INVALID_ARGUMENT
    for kw in ({"num_tokens": -1}, {"heads": -1}, {"head_dim": 12}, {"page_size": 0}, {"page_size": 1 << 24, "num_pages": 128},
               {"k": None}, {"v_cache": None}, {"slots": None}, {"k": 8}, {"slots": 20}, {"k_stride_t": 12},
               {"v_page_stride": -8}):
        refused(lib.fa_append_kv_paged, a, **kw)
    for kw in ({"num_tokens": 0}, {"num_pages": 0}, {"heads": 0}):  # nothing to do
        q = type(a).from_buffer_copy(a)
        for name, value in kw.items():
            setattr(q, name, value)
        assert lib.fa_append_kv_paged(q, x) == _hip.FA_OK


def test_native_functions_hand_on_what_they_do_not_serve():
    import ctypes

    from fused_attn import _hip

    assert _hip._native is not None, "libfused_attn_torch.so is not built"
    n = _hip.NativeFunctions(ctypes.PyDLL(_hip._native._name))
    t = torch.zeros(2, 2, dtype=torch.int32)
    for other in (t, 1, None, "x"):  # tensors of the CPU, and what is no tensor
        assert n.append_kv_paged(other, t, t, t, t) is None
        assert n.allocate_pages(t, other, t, t, t, 16, 1) is None
        assert n.release_pages(t, t, t, t, other, None, 16) is None
        assert n.shared_prefix(t, t, t, t, other, None, None, None, None, 64, 64, False, 0.1, 0) is None
    for number in (1.5, 1 << 70, "x", None):  # no whole numbers, and one past 64 bits
        assert n.allocate_pages(t, t, t, t, t, number, 1) is None
        assert n.shared_prefix(t, t, t, t, t, None, None, None, None, 64, number, False, 0.1, 0) is None
    for f in vars(n).values():
        with pytest.raises(TypeError, match="arguments"):
            f(t)
