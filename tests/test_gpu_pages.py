"""Pages on the GPU: the HIP kernels against the oracle, whole numbers and copied rows bit for bit."""
import pytest
import torch

import fused_attn
from oracle import pages_oracle
from pages_helpers import ALLOCATE, RELEASE, append_oracle, check_allocate, check_release, ints, requests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ALLOCATE, ids=str)
@pytest.mark.parametrize("seed", [0, 1])
def test_allocate(case, seed):
    check_allocate(case, "cuda", seed=seed, wide=seed)


@pytest.mark.parametrize("case", RELEASE, ids=str)
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
def test_release(case, dtype):
    check_release(case, "cuda", dtype=dtype)


def test_sums_past_32_bits_refuse_and_do_not_wrap():
    """Lengths whose sums pass 2^31 and 2^32: the requests that fit before them are served, the others refused."""
    big = 2 ** 31 - 1
    seqlens, new_lens = [3, big, 5, 0, 7], [2, big, big, big, 1]
    table, free = [[i, 90 + i] for i in range(5)], [50, 51, 52]
    t, f = ints(table, "cuda"), ints(free, "cuda")
    got = fused_attn.allocate_pages(t, ints(seqlens, "cuda"), ints(new_lens, "cuda"), f, ints([3], "cuda"), 4, 10)
    want = pages_oracle.allocate(table, seqlens, new_lens, free, 3, 4, 10)
    assert t.tolist() == want[0]
    assert [x.tolist() for x in got] == [*want[1:4], [want[4]]]
    assert want[3] == [5, big, 5, 0, 7]


def test_num_free_out_of_range_is_held_to_the_list():
    for num_free in (-3, 99):
        table, seqlens, new_lens, free, _, tokens = requests((7, 9, 16, 60, 20, 1.0, 0))
        t = ints(table, "cuda")
        got = fused_attn.allocate_pages(t, ints(seqlens, "cuda"), ints(new_lens, "cuda"), ints(free, "cuda"),
                                        ints([num_free], "cuda"), 16, tokens)
        want = pages_oracle.allocate(table, seqlens, new_lens, free, num_free, 16, tokens)
        assert t.tolist() == want[0] and [x.tolist() for x in got] == [*want[1:4], [want[4]]]


def test_strided_lengths_and_transposed_table():
    table, seqlens, new_lens, free, num_free, tokens = requests((33, 9, 16, 60, 20, 1.0, 0))
    wide = lambda v: ints([x for y in v for x in (y, 77)], "cuda")[::2]  # noqa: E731
    t = ints(table, "cuda")
    got = fused_attn.allocate_pages(t, wide(seqlens), wide(new_lens), ints(free, "cuda"), ints([num_free], "cuda"), 16, tokens)
    want = pages_oracle.allocate(table, seqlens, new_lens, free, num_free, 16, tokens)
    assert t.tolist() == want[0] and [x.tolist() for x in got] == [*want[1:4], [want[4]]]
    # a table that is written in place cannot be copied; one that is only read can
    turned = t.t().contiguous().t()
    with pytest.raises(RuntimeError, match="in place"):
        fused_attn.allocate_pages(turned, ints(seqlens, "cuda"), ints(new_lens, "cuda"), ints(free, "cuda"),
                                  ints([num_free], "cuda"), 16, tokens)
    lens, pages = got[2], ints(free + [-1] * 400, "cuda")
    out = fused_attn.release_pages(turned, lens, torch.ones(33, dtype=torch.bool, device="cuda"), pages, got[3], 16)
    want = pages_oracle.release(t.tolist(), lens.tolist(), [True] * 33, free + [-1] * 400, want[4], 16)
    assert pages.tolist() == want[0] and out[0].tolist() == want[1] and out[1].tolist() == [want[2]]


# tokens, heads, D, page
APPEND = [(1, 1, 8, 1), (1, 8, 128, 16), (5, 3, 72, 16), (64, 8, 128, 16), (1000, 2, 64, 48), (777, 4, 256, 32), (4001, 8, 128, 64),
          (300, 16, 40, 7)]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("layout", ["pool", "page_first", "views"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append(case, layout, dtype):
    t, h, d, page = case
    g = torch.Generator(device="cuda").manual_seed(t)
    pages = -(-t // page) + 3
    k, v = (torch.randn(t, h, d, device="cuda", generator=g).to(dtype) for _ in "kv")
    if layout == "page_first":  # pools [num_pages, page_size, Hkv, D], rows of a fused projection
        both = torch.randn(t, 2, h, d, device="cuda", generator=g).to(dtype)
        k, v = both[:, 0], both[:, 1]
        pools = [torch.randn(pages, page, h, d, device="cuda", generator=g).to(dtype).transpose(1, 2) for _ in "kv"]
    elif layout == "views":  # unaligned rows (copied first), K and V halves of one pool
        k = torch.randn(t, h, d + 1, device="cuda", generator=g).to(dtype)[..., 1:]
        both = torch.randn(pages, 2, h, page, d, device="cuda", generator=g).to(dtype)
        pools = [both[:, 0], both[:, 1]]
    else:
        pools = [torch.randn(pages, h, page, d, device="cuda", generator=g).to(dtype) for _ in "kv"]
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:t]
    slots[t // 2] = -1
    if t > 4:
        slots[1], slots[2], slots[3] = pages * page, 2 ** 33, -2 ** 62
    want = append_oracle(k, v, *pools, slots)
    fused_attn.append_kv_paged(k, v, *pools, slots)
    for got, w in zip(pools, want):
        assert torch.equal(got.cpu(), w)


def test_append_special_values_and_repeated_rows():
    """Bits are copied, NaN payloads among them; a row that is broadcast over tokens and heads is read as it is."""
    bits = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(64, 8, 128)
    pools = [torch.zeros(5, 8, 16, 128, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    row = bits[3:4, 1:2].expand(64, 8, 128)
    fused_attn.append_kv_paged(bits, row, *pools, torch.arange(10, 74, device="cuda"))
    got = pools[0].transpose(1, 2).reshape(80, 8, 128).view(torch.int16)
    assert torch.equal(got[10:74], bits.view(torch.int16)) and (got[:10] == 0).all() and (got[74:] == 0).all()
    got = pools[1].transpose(1, 2).reshape(80, 8, 128).view(torch.int16)
    assert torch.equal(got[10:74], row.view(torch.int16).contiguous())


def test_append_behind_4_gib():
    """Offsets past 2^31 elements of a pool."""
    pages = 2 ** 31 // (8 * 64 * 128) + 9
    pools = [torch.zeros(pages, 8, 64, 128, device="cuda", dtype=torch.float16) for _ in "kv"]
    k = torch.randn(130, 8, 128, device="cuda").half()
    slots = (pages - 3) * 64 + torch.arange(130, device="cuda")
    fused_attn.append_kv_paged(k, -k, *pools, slots)
    for pool, x in zip(pools, (k, -k)):
        assert torch.equal(pool[-3:].transpose(1, 2).reshape(192, 8, 128)[:130], x)
        assert not pool[:-3].any() and not pool[-3:].transpose(1, 2).reshape(192, 8, 128)[130:].any()
    del pools


def test_empty():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    slots, cu, lens, left = fused_attn.allocate_pages(i(0, 4), i(0), i(0), i(0), i(()), 16, 0)
    assert slots.shape == (0,) and cu.tolist() == [0] and lens.shape == (0,) and left.shape == () and left == 0
    lens, left = fused_attn.release_pages(i(0, 4), i(0), torch.zeros(0, dtype=torch.bool, device="cuda"), i(3), i(1) + 2, 16)
    assert lens.shape == (0,) and left.tolist() == [2]
    pool = torch.ones(2, 2, 4, 8, device="cuda").half()
    fused_attn.append_kv_paged(pool[:0, :, 0], pool[:0, :, 0], pool, pool.clone(), torch.zeros(0, dtype=torch.int64, device="cuda"))
    fused_attn.append_kv_paged(pool[:, :, 0], pool[:, :, 0], pool[:0], pool[:0], torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert (pool == 1).all()


def test_captured_steps_and_another_stream():
    """A serving step in a graph: lengths, table and list carry over on the device, every replay checked."""
    b, cols, page, steps = 37, 12, 16, 6
    table, seqlens = [[-1] * cols for _ in range(b)], [0] * b
    free, num_free = list(range(500)), 500
    new_lens = [5 + i % 13 for i in range(b)]
    tokens = sum(new_lens)
    t, lens, f, left = ints(table, "cuda"), ints(seqlens, "cuda"), ints(free, "cuda"), ints([num_free], "cuda")
    new = ints(new_lens, "cuda")
    done = torch.tensor([i % 5 == 0 for i in range(b)], device="cuda")
    pools = [torch.zeros(500, 2, page, 64, device="cuda").half() for _ in "kv"]
    k = torch.randn(tokens, 2, 64, device="cuda").half()

    def step():
        slots, cu, grown, n = fused_attn.allocate_pages(t, lens, new, f, left, page, tokens)
        fused_attn.append_kv_paged(k, k, *pools, slots)
        kept, m = fused_attn.release_pages(t, grown, done, f, n, page)
        lens.copy_(kept)
        left.copy_(m)
        return slots

    keep = [x.clone() for x in (t, lens, f, left, *pools)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()  # warms up
        for x, y in zip((t, lens, f, left, *pools), keep):
            x.copy_(y)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots = step()
    want_pools = [p.cpu() for p in pools]
    for _ in range(steps):
        k.copy_(torch.randn_like(k))
        graph.replay()
        table, want, _, grown, num_free = pages_oracle.allocate(table, seqlens, new_lens, free, num_free, page, tokens)
        free, seqlens, num_free = pages_oracle.release(table, grown, done.tolist(), free, num_free, page)
        assert slots.tolist() == want and t.tolist() == table and lens.tolist() == seqlens
        assert f.tolist() == free and left.tolist() == [num_free]
        want_pools = append_oracle(k, k, *want_pools, slots)
        assert all(torch.equal(p.cpu(), w) for p, w in zip(pools, want_pools))
