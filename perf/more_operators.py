"""Operators of a paged K/V cache that requests share, in plain form and through the library.

``kind`` names the operator:

* ``allocate``  ``allocate_pages`` gives a batch's new tokens their pages and slots, on the GPU, from the requests'
  lengths and a list of free pages;
* ``release``   ``release_pages`` puts the pages of finished requests back on that list;
* ``append``    ``append_kv_paged`` writes packed K/V rows at their slots of 16-bit pools;
* ``shared``    ``attention_shared_prefix``: attention over pages for requests that share the start of their context,
  whose keys are read once for all of them.

With ``own`` false, ``run`` computes them with elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8_BLOCK = 64  # keys of an FP8 pool that share a scale

# No drawn workload costs more than the largest listed ones.
MAX_TOKENS = 1 << 18
MAX_APPEND = 65536 * 8 * 128
MAX_FLOPS = 4 * 64 * 128 * 128 * 33500.0
MAX_POOL = 3e8  # values of a pool
MAX_SCORES = 3.2e8  # values of the score matrices that the plain form holds


def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-attention-kernels_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fused_attn

    return fused_attn


# ---------------------------------------------------------------------------------------------------------
# workloads
# ---------------------------------------------------------------------------------------------------------


def _allocate(name, b, held, new, page, room, mix):
    """``b`` requests with up to ``held`` keys get up to ``new`` tokens (1: exactly one each); the list of free pages
    has ``room`` times what they need."""
    return {"name": name, "kind": "allocate", "b": b, "held": held, "new": new, "page": page, "room": room, "mix": mix}


def _release(name, b, held, shared, page, done, mix):
    """A share ``done`` of ``b`` requests with up to ``held`` keys, of which the first ``shared`` stay, has finished."""
    return {"name": name, "kind": "release", "b": b, "held": held, "shared": shared, "page": page, "done": done, "mix": mix}


def _append(name, tokens, hkv, d, dtype, page, mix):
    return {"name": name, "kind": "append", "tokens": tokens, "hkv": hkv, "d": d, "dtype": dtype, "page": page, "mix": mix}


def _shared(name, groups, prefixes, suffix, hq, hkv, nq, d, dtype, cache, causal, page, mix):
    """Groups of ``groups[i]`` requests (texts of numbers: "16,16") behind ``prefixes[i]`` shared keys, each with up to
    ``suffix`` keys of its own."""
    return {"name": name, "kind": "shared", "groups": groups, "prefixes": prefixes, "suffix": suffix, "hq": hq, "hkv": hkv,
            "nq": nq, "d": d, "dtype": dtype, "cache": cache, "causal": causal, "page": page, "mix": mix}


def listed():
    return [
        # one decode step of a serving batch: every request gets one token, few a new page
        _allocate("allocate_b64_decode", 64, 4000, 1, 16, 2.0, 1),
        # prompts of every length arrive beside running requests
        _allocate("allocate_b512_prompts", 512, 3000, 1000, 16, 1.1, 2),
        # a few requests of a batch have finished
        _release("release_b64", 64, 2000, 512, 16, 0.1, 3),
        # many long ones at once
        _release("release_b1024_long", 1024, 16000, 0, 16, 0.6, 4),
        # one decode step's keys and values
        _append("append_64_tokens", 64, 8, 128, "bf16", 16, 5),
        # those of a batch of prompts
        _append("append_40001_tokens", 40001, 8, 128, "bf16", 64, 6),
        # a few requests behind a short system prompt: latency
        _shared("shared_b8_p1000_s100", "8", "992", 100, 32, 8, 1, 128, "fp16", "16bit", False, 16, 7),
        # a serving batch behind a long one
        _shared("shared_b64_p8192_s512", "64", "8192", 512, 32, 8, 1, 128, "bf16", "16bit", True, 64, 8),
        # many short answers at the small head dim, a prefix that ends inside a tile
        _shared("shared_b256_p4080_s1000", "256", "4080", 1000, 64, 8, 1, 64, "fp16", "16bit", True, 16, 9),
        # verifying 4 drafted tokens behind a document
        _shared("shared_b32_q4_p16384_s2000", "32", "16384", 2000, 32, 8, 4, 128, "bf16", "16bit", True, 32, 10),
        # several prompts in one batch, one request without a shared one
        _shared("groups_b49_d256", "16,24,8,1", "4992,704,9984,0", 700, 16, 4, 1, 256, "bf16", "16bit", True, 64, 11),
        # an FP8 cache: parallel answers to one very long document
        _shared("shared_fp8_b128_p32768_s700", "128", "32768", 700, 64, 8, 1, 128, "bf16", "fp8", True, 64, 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more workload of the same ranges."""
    kind = rng.choice(["allocate", "release", "append", "shared", "shared", "shared"])
    mix, page = rng.randrange(1, 1000), rng.choice([16, 16, 32, 48, 64, 256])
    while True:
        if kind == "allocate":
            b, new = _log(rng, 1, 1024), rng.choice([1, 1, 5, _log(rng, 10, 4000)])
            if b * new <= MAX_TOKENS:  # (half the pages: the later requests of a batch get none)
                room = rng.choice([0.5, 1.0, 1.5]) if b >= 16 else rng.choice([1.0, 1.5])
                return _allocate("", b, rng.choice([0, _log(rng, 10, 8000)]), new, page, room, mix)
        elif kind == "release":
            held = _log(rng, 10, 16000)
            return _release("", _log(rng, 1, 1024), held, rng.choice([0, rng.randint(0, held)]), page, rng.random(), mix)
        elif kind == "append":
            tokens, hkv, d = _log(rng, 1, 60000), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 128, 256])
            if tokens * hkv * d <= MAX_APPEND:
                return _append("", tokens, hkv, d, rng.choice(["bf16", "fp16"]), page, mix)
        else:
            hkv, group, d = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 8]), rng.choice([64, 128, 128, 256])
            nq, suffix = rng.choice([1, 1, 1, 2, 4, 7]), _log(rng, 1, 3000)
            cache = rng.choice(["16bit", "16bit", "fp8"])
            if cache == "fp8":
                page = rng.choice([64, 128, 256])
            count = rng.choice([1, 1, 1, 2, 5])
            groups = [_log(rng, 1, 256 // count) for _ in range(count)]
            prefixes = [_log(rng, 100, 33000) // page * page for _ in range(count)]
            b, keys = sum(groups), sum(prefixes)
            rows = hkv * group * nq
            scores = rows * (sum(g * p for g, p in zip(groups, prefixes)) + b * suffix)
            # (a causal request has a key for each of its queries)
            if hkv * d * (keys + b * (suffix + nq + page)) <= MAX_POOL and scores <= MAX_SCORES and 4 * d * scores <= MAX_FLOPS:
                return _shared("", ",".join(map(str, groups)), ",".join(map(str, prefixes)), suffix, hkv * group, hkv, nq, d,
                               rng.choice(["bf16", "fp16"]), cache, rng.random() < 0.7, page, mix)


def _numbers(text):
    return [int(x) for x in text.split(",")]


def _request_lengths(c):
    """(keys held, tokens that arrive) of every request of ``allocate`` and ``release``."""
    rng = random.Random(c["mix"])
    held = [rng.randint(0, c["held"]) for _ in range(c["b"])]
    if c["kind"] == "release":
        return held, [0] * c["b"]
    # prompts arrive for half of the requests, the others go on with one token
    return held, [1 if c["new"] == 1 or rng.random() < 0.5 else rng.randint(1, c["new"]) for _ in held]


def _finished(c):
    rng = random.Random(c["mix"] + 1)
    return [i == 0 or rng.random() < c["done"] for i in range(c["b"])]


def _suffixes(c):
    """Keys of every request behind its prefix, its newest queries' among them; the longest one among them."""
    rng = random.Random(c["mix"])
    b = sum(_numbers(c["groups"]))
    return [c["suffix"] + c["nq"] - 1] + [rng.randint(max(1, c["suffix"] // 16), c["suffix"]) + c["nq"] - 1
                                         for _ in range(b - 1)]


def _cdiv(a, b):
    return -(-a // b)


def work(c):
    if c["kind"] in ("allocate", "release"):
        held, new = _request_lengths(c)
        if c["kind"] == "allocate":
            pages = sum(_cdiv(n + m, c["page"]) - _cdiv(n, c["page"]) for n, m in zip(held, new))
            # lengths in and out, a free page in and its entry of the table out, a slot out
            return {"bytes": 16 * c["b"] + 8 * pages + 8 * sum(new), "flops": 4.0 * (sum(new) + c["b"])}
        pages = sum(max(0, _cdiv(n, c["page"]) - c["shared"] // c["page"]) for n, d in zip(held, _finished(c)) if d)
        return {"bytes": 13 * c["b"] + 8 * pages, "flops": 4.0 * (pages + c["b"])}
    if c["kind"] == "append":
        return {"bytes": c["tokens"] * (8 + 8 * c["hkv"] * c["d"]), "flops": float(c["tokens"])}
    groups, prefixes, suffixes = _numbers(c["groups"]), _numbers(c["prefixes"]), _suffixes(c)
    row = 2 * c["d"] * (2 if c["cache"] == "16bit" else 1)  # of K and of V
    keys = sum(prefixes) + sum(suffixes)
    seen = sum(g * p for g, p in zip(groups, prefixes)) + sum(suffixes)
    return {"bytes": 4 * sum(groups) * c["hq"] * c["nq"] * c["d"] + c["hkv"] * keys * row,
            "flops": 4.0 * c["hq"] * c["nq"] * c["d"] * seen}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(gen, shape, dtype):
    """Rows as a projection gives them: channels of unequal size and offset."""
    d = shape[-1]
    size = torch.exp(0.3 * torch.randn(d, device="cuda", generator=gen))
    shift = 0.3 * torch.randn(d, device="cuda", generator=gen)
    return (torch.randn(shape, device="cuda", generator=gen) * size + shift).to(dtype)


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    page, kind = c["page"], c["kind"]
    s = {"case": c}
    if kind == "append":
        t, hkv, d, dtype = c["tokens"], c["hkv"], c["d"], DTYPES[c["dtype"]]
        pages = _cdiv(t, page) + 64
        s["k"], s["v"] = _rows(gen, (t, hkv, d), dtype), _rows(gen, (t, hkv, d), dtype)
        s["k_cache"], s["v_cache"] = (torch.zeros(pages, hkv, page, d, dtype=dtype, device="cuda") for _ in "kv")
        # runs of a page's slots in scattered pages, as prompts have them; a padding token now and then
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(t, device="cuda") + seed % page
        s["slots"] = order[at // page] * page + at % page
        s["slots"][torch.rand(t, device="cuda", generator=gen) < 0.01] = -1
        return s
    if kind in ("allocate", "release"):
        held, new = _request_lengths(c)
        cols = _cdiv(c["held"] + c.get("new", 0), page) + 1
        have = [_cdiv(n, page) for n in held]
        s["seqlens"], s["new_lens"], s["tokens"] = _ints(held), _ints(new), sum(new)
        if kind == "allocate":
            need = sum(_cdiv(n + m, page) - h for n, m, h in zip(held, new, have))
            free = max(1, int(c["room"] * need))
            spare = 0
        else:
            shared = c["shared"] // page
            s["done"] = torch.tensor(_finished(c), dtype=torch.bool, device="cuda")
            s["keep_lens"] = _ints([c["shared"]] * c["b"])
            free, spare = c["b"], sum(have)
        # (the pool has other users too)
        pages = torch.randperm(sum(have) + free + 4096, device="cuda", generator=gen).to(torch.int32)
        used = torch.arange(cols, device="cuda")[None] < _ints(have)[:, None]
        s["table"] = torch.full((c["b"], cols), -1, dtype=torch.int32, device="cuda")
        s["table"][used] = pages[:sum(have)]
        if kind == "release" and shared:
            s["table"][:, :shared] = torch.where(used[:, :shared], s["table"][:1, :shared], s["table"][:, :shared])
        s["free_pages"] = torch.full((free + spare,), -1, dtype=torch.int32, device="cuda")
        s["free_pages"][:free] = pages[sum(have):sum(have) + free]
        s["num_free"] = _ints([free])
        return s
    groups, prefixes, suffixes = _numbers(c["groups"]), _numbers(c["prefixes"]), _suffixes(c)
    hkv, d, dtype, b = c["hkv"], c["d"], DTYPES[c["dtype"]], sum(groups)
    starts = [p for p, n in zip(prefixes, groups) for _ in range(n)]
    lens = [p + n for p, n in zip(starts, suffixes)]
    cols = max(_cdiv(n, page) for n in lens)
    total = sum(p // page for p in prefixes) + sum(_cdiv(n, page) - p // page for p, n in zip(starts, lens))
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for p, n in zip(prefixes, groups):
        shared = order[at:at + p // page]
        at += len(shared)
        for _ in range(n):
            own_pages = _cdiv(lens[len(table)], page) - len(shared)
            row = shared + order[at:at + own_pages]
            at += own_pages
            table.append(row + [0] * (cols - len(row)))
    s["table"], s["seqlens"] = _ints(table), _ints(lens)
    s["cu_groups"] = _ints([sum(groups[:i]) for i in range(len(groups) + 1)])
    s["prefix_lens"] = _ints(prefixes)
    s["q"] = torch.randn(b, c["hq"], c["nq"], d, device="cuda", generator=gen).to(dtype)
    for name in ("k", "v"):
        if c["cache"] == "16bit":
            s[name + "_cache"], s[name + "_scale"] = _rows(gen, (total, hkv, page, d), dtype), None
            continue
        s[name + "_cache"] = torch.empty(total, hkv, page, d, dtype=torch.float8_e4m3fn, device="cuda")
        s[name + "_scale"] = torch.empty(total, hkv, page // FP8_BLOCK, device="cuda")
        for i in range(0, total, 1024):
            x = _rows(gen, (min(1024, total - i), hkv, page // FP8_BLOCK, FP8_BLOCK, d), torch.float32)
            scale = x.abs().amax((-2, -1)) / 448.0
            s[name + "_scale"][i:i + 1024] = scale
            x8 = (x / scale[..., None, None]).to(torch.float8_e4m3fn)
            s[name + "_cache"].view(torch.uint8)[i:i + 1024] = x8.view(torch.uint8).view(-1, hkv, page, d)
    return s


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------


def _plain_allocate(s):
    c, table, free = s["case"], s["table"], s["num_free"].long()
    page, cols, tokens = c["page"], table.shape[1], s["tokens"]
    n, m = s["seqlens"].long().clamp(min=0), s["new_lens"].long().clamp(min=0)
    end = torch.cumsum(m, 0)
    have, want = (n + page - 1) // page, (n + m + page - 1) // page
    fits = (n + m <= cols * page) & (end <= tokens)
    need = torch.where(fits, want - have, 0)
    ok = fits & ((need == 0) | (torch.cumsum(need, 0) <= free))
    need = torch.where(ok, need, 0)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(cols, device=n.device)
    taken = ok[:, None] & (col >= have[:, None]) & (col < want[:, None])
    at = free - 1 - (first[:, None] + col - have[:, None])
    table.copy_(torch.where(taken, s["free_pages"][at.clamp(0, s["free_pages"].numel() - 1)], table))
    token = torch.arange(tokens, device=n.device)
    seq = torch.searchsorted(end, token, right=True)
    in_batch = seq < n.numel()
    seq = seq.clamp(max=n.numel() - 1)
    pos = n[seq] + token - (end - m)[seq]
    entry = table[seq, (pos // page).clamp(0, cols - 1)].long()
    slots = torch.where(in_batch & ok[seq] & (entry >= 0), entry * page + pos % page, -1)
    cu = torch.cat([torch.zeros_like(end[:1]), end]).clamp(max=tokens).to(torch.int32)
    return {"table": table, "slots": slots, "cu_seqlens": cu, "seqlens": torch.where(ok, n + m, n).to(torch.int32),
            "num_free": (free - need.sum()).to(torch.int32)}


def _plain_release(s):
    c, table, free = s["case"], s["table"], s["num_free"].long()
    page, cols, pages = c["page"], table.shape[1], s["free_pages"]
    n, keep = s["seqlens"].long().clamp(min=0), s["keep_lens"].long().clamp(min=0) // c["page"]
    have = (n + page - 1) // page
    count = torch.where(s["done"], (have - keep).clamp(min=0), 0)
    ok = s["done"] & ((count == 0) | (torch.cumsum(count, 0) + free <= pages.numel()))
    count = torch.where(ok, count, 0)
    first = torch.cumsum(count, 0) - count
    col = torch.arange(cols, device=n.device)
    given = (col >= keep[:, None]) & (col < (keep + count)[:, None])
    at = free + first[:, None] + col - keep[:, None]
    pages[at[given]] = table[given]
    return {"free_pages": pages, "seqlens": torch.where(ok, 0, n).to(torch.int32),
            "num_free": (free + count.sum()).to(torch.int32)}


def _plain_append(s):
    page = s["case"]["page"]
    at = s["slots"]
    keep = (at >= 0) & (at < s["k_cache"].shape[0] * page)
    at = at[keep]
    for name in ("k", "v"):
        s[name + "_cache"][at // page, :, at % page] = s[name][keep]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _keys(s, name, pages, offsets):
    """Rows at (page, offset) of a pool, in 32 bits: pages, offsets [..., N] -> [..., N, Hkv, D]."""
    x = s[name + "_cache"]
    if s[name + "_scale"] is None:
        return x[pages, :, offsets].float()
    x = x.view(torch.uint8)[pages, :, offsets].view(torch.float8_e4m3fn).float()
    return x * s[name + "_scale"][pages, :, offsets // FP8_BLOCK][..., None]


def _plain_shared(s):
    """The prefix's scores for all requests of a group in one product, those behind it padded to the longest."""
    c = s["case"]
    page, hkv, nq, d = c["page"], c["hkv"], c["nq"], c["d"]
    group, scale = c["hq"] // hkv, 1.0 / math.sqrt(d)
    out, b0 = torch.empty(s["q"].shape, device="cuda"), 0
    suffixes = _suffixes(c)
    for n, prefix in zip(_numbers(c["groups"]), _numbers(c["prefixes"])):
        q = s["q"][b0:b0 + n].float().reshape(n, hkv, group * nq, d) * scale
        rows = q.transpose(0, 1).reshape(hkv, n * group * nq, d)
        table, lens = s["table"][b0:b0 + n].long(), s["seqlens"][b0:b0 + n].long()
        pos = torch.arange(prefix, device="cuda")
        kp, vp = (_keys(s, x, table[0, pos // page], pos % page).transpose(0, 1).contiguous() for x in "kv")
        logits = torch.bmm(rows, kp.transpose(1, 2).contiguous()).view(hkv, n, group * nq, prefix).transpose(0, 1)
        width = max(suffixes[b0:b0 + n])
        pos = (prefix + torch.arange(width, device="cuda")).expand(n, width)
        pages = torch.gather(table, 1, (pos // page).clamp(max=table.shape[1] - 1))
        ks, vs = (_keys(s, x, pages, pos % page).transpose(1, 2).contiguous() for x in "kv")
        logits = torch.cat([logits, torch.matmul(q, ks.transpose(2, 3).contiguous())], -1)
        last = lens[:, None].expand(n, nq) - 1
        if c["causal"]:
            last = last - (nq - 1) + torch.arange(nq, device="cuda")
        key = torch.arange(prefix + width, device="cuda")
        seen = (key <= last[..., None]).repeat(1, group, 1)[:, None]
        logits = logits.masked_fill(~seen, -math.inf)
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        # (a masked key's weight is 0, and what lies behind a request's keys in its last page may be anything)
        vs = vs * (pos < lens[:, None])[:, None, :, None]
        shared = torch.bmm(p[..., :prefix].transpose(0, 1).reshape(hkv, n * group * nq, prefix), vp)
        o = shared.view(hkv, n, group * nq, d).transpose(0, 1) + torch.matmul(p[..., prefix:], vs)
        out[b0:b0 + n] = o.reshape(n, c["hq"], nq, d)
        b0 += n
    return out.to(s["q"].dtype)


def _plain(s):
    return {"allocate": _plain_allocate, "release": _plain_release, "append": _plain_append,
            "shared": _plain_shared}[s["case"]["kind"]](s)


def _call(s):
    """The library's calls."""
    lib, c = _library(), s["case"]
    kind = c["kind"]
    if kind == "allocate":
        slots, cu, seqlens, num_free = lib.allocate_pages(s["table"], s["seqlens"], s["new_lens"], s["free_pages"],
                                                          s["num_free"], c["page"], s["tokens"])
        return {"table": s["table"], "slots": slots, "cu_seqlens": cu, "seqlens": seqlens, "num_free": num_free}
    if kind == "release":
        seqlens, num_free = lib.release_pages(s["table"], s["seqlens"], s["done"], s["free_pages"], s["num_free"], c["page"],
                                              keep_lens=s["keep_lens"])
        return {"free_pages": s["free_pages"], "seqlens": seqlens, "num_free": num_free}
    if kind == "append":
        lib.append_kv_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    prefixes, suffix = _numbers(c["prefixes"]), c["suffix"] + c["nq"] - 1
    one = len(prefixes) == 1
    return lib.attention_shared_prefix(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seqlens"],
                                       prefixes[0] if one else s["prefix_lens"], None if one else s["cu_groups"],
                                       causal=c["causal"], max_prefix_len=max(prefixes), max_suffix_len=suffix,
                                       k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(s):
    return _call(s) if own else _plain(s)


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------


def exact(c, seed):
    if c["kind"] in ("allocate", "release"):
        return None  # whole numbers
    s = prepare(c, seed)
    if c["kind"] == "append":
        out = {}
        for name in ("k", "v"):
            pool = s[name + "_cache"].double().transpose(1, 2)  # [page, offset, head, D]: a slot is a row
            rows = pool.reshape(-1, c["hkv"], c["d"])
            taken = torch.nonzero(s["slots"] >= 0)[:, 0]
            rows[s["slots"][taken]] = s[name][taken].double()
            out[name + "_cache"] = rows.view(pool.shape).transpose(1, 2).contiguous()
        return out
    page, hkv, nq, d = c["page"], c["hkv"], c["nq"], c["d"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["seqlens"].tolist()):
        pages = s["table"][i, :_cdiv(n, page)].long()
        kv = []
        for name in ("k", "v"):
            x, scale = s[name + "_cache"][pages], s[name + "_scale"]
            x = x.double() if scale is None else x.double() * scale[pages].double().repeat_interleave(FP8_BLOCK, 2)[..., None]
            kv.append(x.transpose(0, 1).reshape(hkv, -1, d)[:, :n])
        q = s["q"][i].double().reshape(hkv, -1, d)
        logits = q @ kv[0].transpose(1, 2).contiguous() * d ** -0.5
        if c["causal"]:
            hidden = torch.ones(nq, n, dtype=torch.bool, device="cuda").triu(n - nq + 1)
            logits = logits.masked_fill(hidden.repeat(logits.shape[1] // nq, 1), -math.inf)
        out[i] = (torch.softmax(logits, -1) @ kv[1]).reshape(c["hq"], nq, d)
    return out
