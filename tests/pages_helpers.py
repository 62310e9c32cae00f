"""Requests and pools shared by the tests of pages."""
import random

import torch

import fused_attn
from oracle import pages_oracle

# b, columns, page, held keys up to, new tokens up to, share of the pages needed that are free, tokens too few by
ALLOCATE = [
    (1, 1, 1, 0, 1, 1.0, 0),
    (1, 4, 16, 30, 1, 1.0, 0),
    (3, 5, 16, 48, 20, 1.0, 0),
    (7, 9, 48, 200, 300, 2.0, 0),
    (64, 40, 16, 500, 1, 1.0, 0),
    (65, 40, 16, 500, 90, 0.5, 0),  # too few pages: later requests are refused
    (65, 20, 16, 500, 90, 1.0, 0),  # rows too narrow for some
    (33, 30, 7, 100, 60, 1.0, 50),  # more tokens than the caller has room for
    (33, 30, 7, 100, 60, 1.0, -300),  # fewer: the rest belong to no request
    (1023, 6, 64, 200, 3, 0.9, 0),
    (1024, 6, 64, 200, 3, 1.0, 0),
    (1025, 6, 64, 200, 3, 1.0, 0),
    (3100, 4, 32, 60, 40, 0.8, 7),
    (0, 3, 16, 0, 0, 1.0, -5),
    (5, 0, 16, 0, 4, 1.0, 0),  # no columns: only requests without tokens fit
    (4, 300, 256, 60000, 9000, 1.0, 0),
]
RELEASE = [  # b, columns, page, held keys up to, share finished, shared keys, room for so many pages too few
    (1, 1, 1, 1, 1.0, 0, 0),
    (3, 5, 16, 80, 0.6, 0, 0),
    (64, 40, 16, 640, 0.3, 64, 0),
    (65, 40, 7, 280, 0.9, 30, 25),  # the list is too short for some
    (33, 10, 16, 300, 1.0, 0, 0),  # lengths beyond a row's columns
    (1025, 6, 64, 380, 0.5, 0, 0),
    (3100, 4, 32, 128, 0.7, 33, 100),
    (300, 500, 16, 8000, 1.0, 0, 0),
    (0, 3, 16, 0, 1.0, 0, 0),
    (9, 12, 16, 190, 0.0, 0, 0),
]


def requests(case, seed=0):
    """Lists (table, seqlens, new_lens, free_pages, num_free, num_tokens) of an ALLOCATE case."""
    b, cols, page, held, new, share, short = case
    rng = random.Random(seed)
    seqlens = [rng.randint(0, min(held, cols * page)) for _ in range(b)]
    new_lens = [rng.choice([0, 1, rng.randint(0, new)]) for _ in range(b)]
    if b > 4:
        seqlens[2], new_lens[3] = -5, -2  # read as 0
    need = sum(-(-(max(n, 0) + max(m, 0)) // page) - -(-max(n, 0) // page) for n, m in zip(seqlens, new_lens))
    ids = rng.sample(range(10 * (b * cols + need + 8)), b * cols + need + 8)
    table = [[ids.pop() for _ in range(cols)] for _ in range(b)]
    if b > 4 and cols:
        table[4][0] = -1  # a page nobody has
    num_free = int(share * need)
    free_pages = [ids.pop() for _ in range(num_free + 3)]
    return table, seqlens, new_lens, free_pages, num_free, max(0, sum(max(m, 0) for m in new_lens) - short)


def finished(case, seed=0):
    """Lists (table, seqlens, done, free_pages, num_free, keep_lens) of a RELEASE case."""
    b, cols, page, held, share, shared, short = case
    rng = random.Random(seed)
    seqlens = [rng.randint(0, held) for _ in range(b)]
    done = [rng.random() < share for _ in range(b)]
    keep = [rng.randint(0, 2 * shared) for _ in range(b)] if shared else None
    if b > 4:
        seqlens[2] = -5
    ids = rng.sample(range(10 * (b * cols + 8)), b * cols + 8)
    table = [[ids.pop() for _ in range(cols)] for _ in range(b)]
    _, _, count = pages_oracle.release(table, seqlens, done, [0] * (b * cols + 5), 5, page, keep)
    free_pages = [ids.pop() for _ in range(5)] + [-7] * max(0, count - 5 - short)
    return table, seqlens, done, free_pages, 5, keep


def ints(values, device, shape=None):
    t = torch.tensor(values, dtype=torch.int32, device=device)
    return t if shape is None else t.reshape(shape)


def check_allocate(case, device, seed=0, wide=0):
    """allocate_pages against the oracle; ``wide``: columns of the table's buffer behind its own, which stay as they are."""
    table, seqlens, new_lens, free_pages, num_free, tokens = requests(case, seed)
    b, cols, page = case[:3]
    buffer = torch.full((b, cols + wide), -99, dtype=torch.int32, device=device)
    buffer[:, :cols] = ints(table, device, (b, cols))
    free = ints(free_pages, device)
    lens, new = ints(seqlens, device), ints(new_lens, device)
    got = fused_attn.allocate_pages(buffer[:, :cols], lens, new, free, ints([num_free], device), page, tokens)
    want = pages_oracle.allocate(table, seqlens, new_lens, free_pages, num_free, page, tokens)
    assert got[0].dtype == torch.int64 and all(t.dtype == torch.int32 for t in got[1:])
    assert buffer[:, :cols].tolist() == want[0]
    assert (buffer[:, cols:] == -99).all()
    assert got[0].tolist() == want[1]
    assert got[1].tolist() == want[2]
    assert got[2].tolist() == want[3]
    assert got[3].tolist() == [want[4]]
    assert free.tolist() == free_pages and lens.tolist() == seqlens and new.tolist() == new_lens


def check_release(case, device, seed=0, dtype=torch.bool):
    table, seqlens, done, free_pages, num_free, keep = finished(case, seed)
    b, cols, page = case[:3]
    t, free, lens = ints(table, device, (b, cols)), ints(free_pages, device), ints(seqlens, device)
    got = fused_attn.release_pages(t, lens, torch.tensor(done, dtype=dtype, device=device), free,
                                   ints([num_free], device), page, keep_lens=None if keep is None else ints(keep, device))
    want = pages_oracle.release(table, seqlens, done, free_pages, num_free, page, keep)
    assert free.tolist() == want[0]
    assert got[0].tolist() == want[1] and got[1].tolist() == [want[2]]
    assert t.tolist() == table and lens.tolist() == seqlens


def append_oracle(k, v, k_cache, v_cache, slots):
    """Copies of the pools (on the CPU) with the rows written one at a time."""
    pools = []
    for x, pool in ((k, k_cache), (v, v_cache)):
        x, pool = x.cpu(), pool.cpu().clone()
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pool.shape[0] * pool.shape[2]:
                pool[slot // pool.shape[2], :, slot % pool.shape[2]] = x[t]
        pools.append(pool)
    return pools
