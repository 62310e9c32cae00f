"""Paged caches whose requests share prefixes, and the check against attention in 64 bits (tests of shared prefixes)."""
import math

import torch

import fused_attn
from cache_norms import check_rows
from oracle import cache_oracle as cor


class Case:
    """Groups of requests behind shared keys.

    ``lens``: all keys of each request (shorter than its prefix, or 0, allowed).  The rows of a group name the same pages
    for the whole pages of the prefix, and copies for the rest.  What no request holds is NaN: unused pages, rows behind a
    request's keys; a table entry behind them is out of the pool or names an unused page."""

    def __init__(self, groups, prefixes, lens, hkv=2, d=64, page=16, dtype=torch.bfloat16, fp8=False, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        b = sum(groups)
        assert len(lens) == b
        n = max(max(lens), 1)
        cols = -(-n // page) + 1
        make = lambda *s: torch.randn(*s, device=device, generator=g) * torch.exp(  # noqa: E731
            0.5 * torch.randn(s[-1], device=device, generator=g))
        start = [p for p, c in zip(prefixes, groups) for _ in range(c)]
        group_of = [i for i, c in enumerate(groups) for _ in range(c)]
        # (nobody longer than the prefix: the last page that the longest request has is shared too, since an FP8 page's scales
        # depend on all its rows, and copies with other rows behind would hold other keys)
        most = [max([lens[i] for i in range(b) if group_of[i] == gi], default=0) for gi in range(len(groups))]
        shared_pages = [p // page if m > p else -(-m // page) for p, m in zip(prefixes, most)]
        total = sum(shared_pages) + sum(max(0, -(-lens[i] // page) - shared_pages[group_of[i]]) for i in range(b)) + 3
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        shared = [[order.pop() for _ in range(c)] for c in shared_pages]
        self.kv, pools, scales = [], [], []
        for _ in "kv":
            x = make(b, hkv, n, d)
            for i in range(b):  # the group's keys are its first request's
                x[i, :, :start[i]] = x[group_of.index(group_of[i]), :, :start[i]]
            x = x.to(dtype)
            self.kv.append(x.double())
            pools.append(torch.full((total, hkv, page, d), math.nan, dtype=dtype, device=device))
        table = torch.full((b, cols), -1, dtype=torch.int32)
        for i in range(b):
            held = -(-lens[i] // page)
            row = shared[group_of[i]][:held]
            row += [order.pop() for _ in range(held - len(row))]
            table[i, :held] = torch.tensor(row, dtype=torch.int32)
            table[i, held:] = order[0] if i % 2 else 2 ** 31 - 1
            for j, at in enumerate(row):
                rows = min(page, lens[i] - j * page)
                for pool, x in zip(pools, self.kv):
                    pool[at, :, :rows] = x[i, :, j * page:j * page + rows].to(dtype)
        self.scales = {}
        if fp8:
            for i, name in enumerate(("k_scale", "v_scale")):
                # a page at a time, so that requests' partial pages are coded by the same rule
                pool = pools[i].nan_to_num(0.0)
                x8, sc = fused_attn.quantize_kv_fp8(pool)
                value = fused_attn.dequantize_kv_fp8(x8, sc).double()
                for r in range(b):
                    held = -(-lens[r] // page)
                    if held:
                        rows = value[table[r, :held].long().to(device)].transpose(0, 1).reshape(hkv, held * page, d)
                        self.kv[i][r, :, :lens[r]] = rows[:, :lens[r]]
                pools[i], self.scales[name] = x8, sc
        self.k, self.v = pools
        self.table = table.to(device)
        self.lens, self.groups, self.prefixes = lens, groups, prefixes
        self.seqlens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.prefix_lens = torch.tensor(prefixes, dtype=torch.int32, device=device)
        cu = [0]
        for c in groups:
            cu.append(cu[-1] + c)
        self.cu_groups = torch.tensor(cu, dtype=torch.int32, device=device)
        self.start = start

    def q(self, hq, nq, dtype=None, seed=1):
        g = torch.Generator(device=self.k.device).manual_seed(seed)
        dtype = self.kv_dtype(dtype)
        return torch.randn(len(self.lens), hq, nq, self.k.shape[3], device=self.k.device, generator=g).to(dtype)

    def kv_dtype(self, dtype):
        return dtype if dtype is not None else self.k.dtype if self.k.dtype != torch.float8_e4m3fn else torch.bfloat16

    def call(self, q, **kw):
        args = dict(self.scales)
        if len(self.groups) > 1:
            args["cu_groups"] = self.cu_groups
        args.update(kw)
        return fused_attn.attention_shared_prefix(q, self.k, self.v, self.table, self.seqlens,
                                                  args.pop("prefix_lens", self.prefix_lens), **args)

    def check(self, got, q, causal=False, lse=None):
        assert got.shape == q.shape and got.dtype == q.dtype
        for i, n in enumerate(self.lens):
            if n == 0:
                assert (got[i] == 0).all()
        worst = check_rows(got, q, *self.kv, causal=causal, lens=self.lens)
        if lse is not None:
            want = cor.attention(q, *self.kv, causal=causal, lens=self.lens)[1]
            assert torch.equal(torch.isneginf(lse), torch.isneginf(want))
            fine = ~torch.isneginf(want)
            # the 16-bit row sum's rounding (each P by at most half a step: q's type) beside the scores' in 32 bits
            tol = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[q.dtype] + 2.0 ** -12
            assert ((lse.double() - want)[fine].abs() <= tol).all()
        return worst
