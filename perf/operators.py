"""Operators of a 4-bit K/V cache and of eviction by attention weight, in plain form and through the library.

``kind`` names the operator:

* ``quantize``  ``quantize_kv_int4`` writes K/V rows as 4-bit codes with an fp16 (scale, zero) pair a row,
  ``dequantize_kv_int4`` reads them back;
* ``append``    ``append_kv_int4`` writes the newest tokens of a serving batch into 4-bit pages;
* ``attend``    ``attention_int4``: attention over a 4-bit cache, dense;
* ``paged``     ``attention_paged`` over 4-bit pools with ragged lengths;
* ``scored``    ``attention_scored``: attention that also adds each key's attention weight to its score, over a
  16-bit or a 4-bit cache;
* ``evict``     ``evict_kv`` keeps the keys of the highest scores and the most recent ones.

With ``own`` false, ``run`` computes them with elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP16_MAX = 65504.0

# No drawn workload costs more than the largest listed ones.
MAX_KEYS = {"quantize": 16 * 8 * 32768 * 128, "attend": 32 * 8 * 32768 * 128, "evict": 16 * 8 * 8192 * 128}
MAX_SCORES = 3.4e7  # values of the score matrix that the plain form holds


def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-attention-kernels_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fused_attn

    return fused_attn


# ---------------------------------------------------------------------------------------------------------
# workloads
# ---------------------------------------------------------------------------------------------------------


def _quantize(name, b, hkv, n, d, dtype, layout="bhnd"):
    return {"name": name, "kind": "quantize", "b": b, "hkv": hkv, "n": n, "d": d, "dtype": dtype, "layout": layout}


def _append(name, b, hkv, nk, new, d, dtype, page, mix):
    return {"name": name, "kind": "append", "b": b, "hkv": hkv, "nk": nk, "new": new, "d": d, "dtype": dtype,
            "page": page, "mix": mix}


def _attend(name, b, hq, hkv, nq, nk, d, dtype, causal, mix=0):
    return {"name": name, "kind": "attend", "b": b, "hq": hq, "hkv": hkv, "nq": nq, "nk": nk, "d": d,
            "dtype": dtype, "causal": causal, "mix": mix}


def _paged(name, b, hq, hkv, nq, nk, d, dtype, causal, page, mix):
    return {"name": name, "kind": "paged", "b": b, "hq": hq, "hkv": hkv, "nq": nq, "nk": nk, "d": d,
            "dtype": dtype, "causal": causal, "page": page, "mix": mix}


def _scored(name, b, hq, hkv, nq, nk, d, dtype, causal, cache, mix=0):
    return {"name": name, "kind": "scored", "b": b, "hq": hq, "hkv": hkv, "nq": nq, "nk": nk, "d": d,
            "dtype": dtype, "causal": causal, "cache": cache, "mix": mix}


def _evict(name, b, hkv, nk, keep, recent, d, dtype, cache, mix=0):
    return {"name": name, "kind": "evict", "b": b, "hkv": hkv, "nk": nk, "keep": keep, "recent": recent, "d": d,
            "dtype": dtype, "cache": cache, "mix": mix}


def listed():
    return [
        # the keys of one short prompt go into the cache: latency
        _quantize("quantize_b1_n1000", 1, 8, 1000, 128, "bf16"),
        # the keys of a batch of long contexts, from the [B, N, H, D] projections: the stream is all there is
        _quantize("quantize_b16_n32768", 16, 8, 32768, 128, "bf16", "bnhd"),
        # one decode step's new tokens of a serving batch, into 16-key pages
        _append("append_b64_new1", 64, 8, 500, 1, 64, "fp16", 16, 5),
        # one interactive request generating a token early in its context
        _attend("attend_b1_ctx1000", 1, 32, 8, 1, 1000, 128, "fp16", True),
        # a serving batch deep into long contexts
        _attend("attend_b32_ctx32768", 32, 32, 8, 1, 32768, 128, "bf16", True),
        # verifying 16 drafted tokens at the largest head dim
        _attend("attend_b8_q16_ctx20000", 8, 32, 8, 16, 20000, 256, "bf16", True),
        # a continuous-batching step: requests of every age, in 16-key pages
        _paged("paged_b48_ragged8k", 48, 64, 8, 1, 8192, 64, "fp16", True, 16, 7),
        # a decode step that scores the keys of a 16-bit cache
        _scored("scored_b16_ctx16384", 16, 32, 8, 1, 16384, 128, "bf16", True, "16bit"),
        # the same over a 4-bit cache, requests of every age
        _scored("scored_int4_b32_ragged8191", 32, 64, 8, 1, 8191, 128, "bf16", True, "int4", 3),
        # the last 32 queries of a prompt score its keys before it is cut down
        _scored("scored_window32_ctx8191", 1, 32, 8, 32, 8191, 128, "fp16", True, "16bit"),
        # a 4-bit cache of a serving batch cut to half
        _evict("evict_int4_b16_8192_to_4096", 16, 8, 8192, 4096, 256, 128, "bf16", "int4", 2),
        # one long prompt's 16-bit cache cut to a quarter
        _evict("evict_b1_65536_to_16384", 1, 8, 65536, 16384, 1024, 128, "bf16", "16bit"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more workload of the same ranges."""
    kind = rng.choice(["quantize", "append", "attend", "attend", "paged", "scored", "scored", "evict"])
    d, dtype, mix = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "fp16"]), rng.randrange(1, 1000)
    while True:
        hkv, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 8])
        b, nk = _log(rng, 1, 64), _log(rng, 100, 66000)
        causal = rng.random() < 0.7
        if kind == "quantize":
            if b * hkv * nk * d <= MAX_KEYS["quantize"]:
                return _quantize("", b, hkv, nk, d, rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["bhnd", "bnhd"]))
        elif kind == "append":
            nk = min(nk, 2000)
            if b * hkv * nk * d <= MAX_KEYS["evict"]:
                return _append("", b, hkv, nk, rng.choice([1, 1, 2, 5]), d, dtype, rng.choice([16, 48, 64]), mix)
        elif kind in ("attend", "paged"):
            nq = rng.choice([1, 1, 1, 2, 4, 7, 16])
            if b * hkv * nk * d <= MAX_KEYS["attend"] / 2 and b * hkv * group * nq * nk <= 4 * MAX_SCORES:
                if kind == "attend":
                    return _attend("", b, hkv * group, hkv, nq, nk, d, dtype, causal, rng.choice([0, mix]))
                return _paged("", b, hkv * group, hkv, nq, nk, d, dtype, causal, rng.choice([16, 32, 48, 64, 256]), mix)
        elif kind == "scored":
            nq = rng.choice([1, 1, 1, 2, 5, 32])
            if b * hkv * nk * d <= MAX_KEYS["attend"] / 4 and b * hkv * group * nq * nk <= 4 * MAX_SCORES:
                return _scored("", b, hkv * group, hkv, nq, nk, d, dtype, causal, rng.choice(["16bit", "int4"]),
                               rng.choice([0, mix]))
        else:
            keep = max(1, int(nk * rng.uniform(0.1, 0.9)))
            if b * hkv * nk * d <= MAX_KEYS["evict"]:
                return _evict("", b, hkv, nk, keep, rng.choice([0, keep // 8, keep // 2]), d, dtype,
                              rng.choice(["16bit", "int4"]), mix)


def _lengths(c):
    """Keys per sequence: of every age in a ragged batch (``mix``), the longest among them."""
    if not c.get("mix"):
        return [c["nk"]] * c["b"]
    rng = random.Random(c["mix"])
    return [c["nk"]] + [rng.randint(max(1, c["nk"] // 12), c["nk"]) for _ in range(c["b"] - 1)]


def work(c):
    d, hkv = c["d"], c["hkv"]
    row4 = d // 2 + 4  # a 4-bit row: its codes, and its scale and zero
    if c["kind"] == "quantize":
        rows = c["b"] * hkv * c["n"]
        size = DTYPES[c["dtype"]].itemsize
        # the rows in, the cache out; the cache in, its values out
        return {"bytes": rows * (2 * size * d + 2 * row4), "flops": 6.0 * rows * d}
    if c["kind"] == "append":
        pages = c["b"] * _columns(c)
        rows = pages * c["page"] * hkv
        # K and V: the new rows in and out, then the pools in and their values out
        return {"bytes": 2 * (c["b"] * hkv * c["new"] * (2 * d + row4) + rows * (row4 + 2 * d)), "flops": 2.0 * 2 * rows * d}
    keys = sum(_lengths(c))
    row = 2 * (row4 if c["kind"] in ("attend", "paged") or c["cache"] == "int4" else 2 * d)  # of K and of V
    if c["kind"] == "evict":
        kept = sum(min(n, c["keep"]) for n in _lengths(c))
        # every score in; of the kept keys the rows in and out, the score and the index out
        return {"bytes": hkv * (4 * keys + kept * (2 * row + 8)), "flops": float(hkv * keys)}
    rows = c["b"] * c["hq"] * c["nq"]
    scores = 8 * hkv * keys if c["kind"] == "scored" else 0
    return {"bytes": 4 * rows * d + hkv * keys * row + scores, "flops": 4.0 * c["hq"] * c["nq"] * d * keys}


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------


def _columns(c):
    return -(-(c["nk"] + c.get("new", 0)) // c["page"])


def _rows(gen, shape, dtype):
    """Rows as a projection gives them: channels of unequal size and offset."""
    d = shape[-1]
    size = torch.exp(0.5 * torch.randn(d, device="cuda", generator=gen))
    shift = 0.5 * torch.randn(d, device="cuda", generator=gen)
    return (torch.randn(shape, device="cuda", generator=gen) * size + shift).to(dtype)


def _encode(x):
    """4-bit codes, two a byte (the even channel in the low half), and (scale, zero) in fp16, a row of x."""
    x = x.float()
    low, high = (y.clamp(-FP16_MAX, FP16_MAX) for y in (x.amin(-1), x.amax(-1)))
    zero, scale = low.half(), ((high - low) * (1.0 / 15.0)).half()
    step, start = scale.float()[..., None], zero.float()[..., None]
    code = torch.round((x - start) / step)
    code = torch.where(step > 0, code, torch.zeros_like(code)).clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([scale, zero], -1)


def _cache(gen, b, hkv, n, d, dtype):
    """A 4-bit cache [B, Hkv, N, D/2] and its (scale, zero) pairs, made a sequence at a time."""
    codes = torch.empty(b, hkv, n, d // 2, dtype=torch.uint8, device="cuda")
    pairs = torch.empty(b, hkv, n, 2, dtype=torch.float16, device="cuda")
    for i in range(b):
        codes[i], pairs[i] = _encode(_rows(gen, (hkv, n, d), dtype))
    return codes, pairs


def _to_pages(x, page, order):
    """[B, Hkv, cols * page, W] -> pools [B * cols, Hkv, page, W] with page ``i`` of the batch at ``order[i]``."""
    b, hkv, n, w = x.shape
    pages = x.view(b, hkv, n // page, page, w).permute(0, 2, 1, 3, 4).reshape(-1, hkv, page, w)
    pool = torch.empty_like(pages)
    pool[order] = pages
    return pool


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype, d, hkv, b = c["kind"], DTYPES[c["dtype"]], c["d"], c["hkv"], c["b"]
    s = {"case": c}
    if kind == "quantize":
        bnhd = c["layout"] == "bnhd"
        x = torch.empty((b, c["n"], hkv, d) if bnhd else (b, hkv, c["n"], d), dtype=dtype, device="cuda")
        for i in range(b):
            x[i] = _rows(gen, x.shape[1:], dtype)
        s["x"] = x.transpose(1, 2) if bnhd else x
        return s
    lens = _lengths(c)
    s["seqlens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if kind in ("append", "paged"):
        cols = _columns(c)
        order = torch.randperm(b * cols, device="cuda", generator=gen)
        s["table"] = order.view(b, cols).to(torch.int32)
        for name in ("k", "v"):
            codes, pairs = _cache(gen, b, hkv, cols * c["page"], d, dtype)
            s[name], s[name + "_scale"] = _to_pages(codes, c["page"], order), _to_pages(pairs, c["page"], order)
        if kind == "append":
            s["new_k"], s["new_v"] = (_rows(gen, (b, hkv, c["new"], d), dtype) for _ in "kv")
    else:
        for name in ("k", "v"):
            if kind == "attend" or c["cache"] == "int4":
                s[name], s[name + "_scale"] = _cache(gen, b, hkv, c["nk"], d, dtype)
            else:
                s[name], s[name + "_scale"] = _rows(gen, (b, hkv, c["nk"], d), dtype), None
    if kind in ("scored", "evict"):
        # weights that earlier steps left: a few keys hold most, many hold none
        w = torch.exp(2.0 * torch.randn(b, hkv, c["nk"], device="cuda", generator=gen))
        s["scores"] = w * (torch.rand(w.shape, device="cuda", generator=gen) > 0.1)
    if kind in ("attend", "paged", "scored"):
        s["q"] = torch.randn(b, c["hq"], c["nq"], d, device="cuda", generator=gen).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------


def _decode(codes, pairs):
    """The values of a 4-bit cache, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return code.float() * pairs[..., :1].float() + pairs[..., 1:].float()


def _values(s, name):
    return s[name].float() if s[name + "_scale"] is None else _decode(s[name], s[name + "_scale"])


def _gathered(pool, table):
    """[P, Hkv, page, W] pools through the block table: [B, Hkv, cols * page, W]."""
    b, cols = table.shape
    x = pool[table.long().reshape(-1)]
    return x.view(b, cols, *x.shape[1:]).transpose(1, 2).reshape(b, x.shape[1], cols * x.shape[2], x.shape[3])


def _softmax_attention(q, k, v, lens, causal):
    """Attention of q [B, Hq, Nq, D] over the first ``lens[b]`` keys of k, v [B, Hkv, N, D]: the output in 32 bits and
    the probabilities [B, Hkv, G * Nq, N].  Causal: the last query sees every key."""
    b, hq, nq, d = q.shape
    hkv, n = k.shape[1:3]
    logits = torch.matmul(q.float().reshape(b, hkv, -1, d), k.transpose(-1, -2)) / math.sqrt(d)
    key = torch.arange(n, device=q.device)
    last = lens.long()[:, None].expand(b, nq) - 1
    if causal:
        last = last - (nq - 1) + torch.arange(nq, device=q.device)
    seen = (key <= last[..., None]).repeat(1, hq // hkv, 1)[:, None]
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, v).reshape(b, hq, nq, d), p


def _kept(scores, lens, keep, recent):
    """Indices [B, Hkv, keep] of the kept keys in ascending order, -1 past them."""
    n = scores.shape[-1]
    key, end = torch.arange(n, device=scores.device), lens.long()[:, None, None]
    rank = torch.where(key >= end - recent, torch.full_like(scores, math.inf), scores)
    rank = torch.where(key >= end, torch.full_like(scores, -math.inf), rank)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.sort(best, dim=-1).values
    return torch.where(best < end, best, torch.full_like(best, -1))


def _rows_of(x, at):
    """Rows ``at`` of x [B, Hkv, N, ...], zeros where it is -1."""
    x3 = x if x.dim() == 4 else x[..., None]
    got = torch.gather(x3, 2, at.clamp(min=0)[..., None].expand(*at.shape, x3.shape[-1]))
    got = torch.where(at[..., None] >= 0, got, torch.zeros_like(got))
    return got if x.dim() == 4 else got[..., 0]


def _plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "quantize":
        codes, pairs = _encode(s["x"])
        return {"values": _decode(codes, pairs).to(s["x"].dtype), "scale": pairs}
    if kind == "append":
        end, page = s["seqlens"].long(), c["page"]
        at = end[:, None] + torch.arange(c["new"], device=end.device)
        pages, slots = torch.gather(s["table"].long(), 1, at // page), at % page
        out = {}
        for name in ("k", "v"):
            codes, pairs = _encode(s["new_" + name])
            s[name][pages, :, slots] = codes.transpose(1, 2)
            s[name + "_scale"][pages, :, slots] = pairs.transpose(1, 2)
            out[name] = _decode(s[name], s[name + "_scale"]).to(DTYPES[c["dtype"]])
        return out
    if kind == "evict":
        at = _kept(s["scores"], s["seqlens"], c["keep"], c["recent"])
        caches = [x for x in (s["k"], s["k_scale"], s["v"], s["v_scale"]) if x is not None]
        return {"caches": [_rows_of(x, at) for x in caches], "scores": _rows_of(s["scores"], at),
                "index": at.to(torch.int32), "seqlens": s["seqlens"].clamp(max=c["keep"])}
    if kind == "paged":
        k, v = (_decode(_gathered(s[x], s["table"]), _gathered(s[x + "_scale"], s["table"])) for x in ("k", "v"))
    else:
        k, v = _values(s, "k"), _values(s, "v")
    o, p = _softmax_attention(s["q"], k, v, s["seqlens"], c["causal"])
    if kind == "scored":
        return {"o": o.to(s["q"].dtype), "scores": s["scores"] + p.sum(2)}
    return o.to(s["q"].dtype)


def _call(s):
    """The library's calls."""
    lib, c = _library(), s["case"]
    kind = c["kind"]
    if kind == "quantize":
        codes, pairs = lib.quantize_kv_int4(s["x"])
        return {"values": lib.dequantize_kv_int4(codes, pairs, s["x"].dtype), "scale": pairs}
    if kind == "append":
        lib.append_kv_int4(s["new_k"], s["new_v"], s["k"], s["k_scale"], s["v"], s["v_scale"], s["seqlens"],
                           block_table=s["table"])
        dtype = DTYPES[c["dtype"]]
        return {x: lib.dequantize_kv_int4(s[x], s[x + "_scale"], dtype) for x in ("k", "v")}
    if kind == "evict":
        caches = [x for x in (s["k"], s["k_scale"], s["v"], s["v_scale"]) if x is not None]
        caches, scores, index, seqlens = lib.evict_kv(s["scores"], caches, c["keep"], recent=c["recent"],
                                                      seqlens_k=s["seqlens"])
        return {"caches": caches, "scores": scores, "index": index, "seqlens": seqlens}
    if kind == "paged":
        return lib.attention_paged(s["q"], s["k"], s["v"], s["table"], s["seqlens"], causal=c["causal"],
                                   max_seqlen_k=c["nk"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "scored":
        o, scores = lib.attention_scored(s["q"], s["k"], s["v"], scores=s["scores"], causal=c["causal"],
                                         seqlens_k=s["seqlens"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"o": o, "scores": scores}
    return lib.attention_int4(s["q"], s["k"], s["k_scale"], s["v"], s["v_scale"], causal=c["causal"],
                              seqlens_k=s["seqlens"] if c["mix"] else None)


def run(s):
    return _call(s) if own else _plain(s)


# ---------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------


def _stands_for(codes, pairs):
    """What 4-bit rows stand for: code * scale + zero, the even channel in a byte's low half."""
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    scale, zero = pairs[..., 0:1].double(), pairs[..., 1:2].double()
    out[..., 0::2] = codes.remainder(16).double() * scale + zero
    out[..., 1::2] = codes.div(16, rounding_mode="floor").double() * scale + zero
    return out


def _nearest(x):
    """x -> (what its 4-bit form stands for, its scale and zero), from 16 levels between a row's ends."""
    x = x.double()
    ends = torch.stack([x.min(-1).values, x.max(-1).values], -1).clamp(-FP16_MAX, FP16_MAX)
    zero = ends[..., 0].half().double()
    scale = ((ends[..., 1] - ends[..., 0]) / 15).half().double()
    level = torch.where(scale[..., None] > 0, (x - zero[..., None]) / scale[..., None], 0.0).round().clamp(0, 15)
    return zero[..., None] + scale[..., None] * level, torch.stack([scale, zero], -1)


def exact(c, seed):
    if c["kind"] == "evict":
        return None  # copies and whole numbers
    s = prepare(c, seed)
    if c["kind"] == "quantize":
        values, pairs = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda"), []
        for i, x in enumerate(s["x"]):
            values[i], pair = _nearest(x)
            pairs.append(pair)
        return {"values": values, "scale": torch.stack(pairs)}
    lens = _lengths(c)
    if c["kind"] == "append":
        out = {}
        for name in ("k", "v"):
            pool = _stands_for(s[name], s[name + "_scale"])
            for i, n in enumerate(lens):
                for j in range(c["new"]):
                    page = int(s["table"][i, (n + j) // c["page"]])
                    pool[page, :, (n + j) % c["page"]] = _nearest(s["new_" + name][i, :, j])[0]
            out[name] = pool
        return out
    group, nq, d = c["hq"] // c["hkv"], c["nq"], c["d"]
    outs, scores = [], s["scores"].double() if c["kind"] == "scored" else None
    for i, n in enumerate(lens):
        kv = []
        for name in ("k", "v"):
            codes, pairs = s[name], s[name + "_scale"]
            if c["kind"] == "paged":
                pages = s["table"][i].long()
                codes, pairs = (x[pages].transpose(0, 1).flatten(1, 2) for x in (codes, pairs))
            else:
                codes, pairs = codes[i], None if pairs is None else pairs[i]
            kv.append(codes[:, :n].double() if pairs is None else _stands_for(codes[:, :n], pairs[:, :n]))
        k, v = (x.repeat_interleave(group, 0) for x in kv)
        logits = s["q"][i].double() @ k.transpose(1, 2).contiguous() * d ** -0.5
        if c["causal"]:
            hidden = torch.ones(nq, n, dtype=torch.bool, device="cuda").triu(n - nq + 1)
            logits = logits.masked_fill(hidden, -math.inf)
        p = torch.softmax(logits, -1).nan_to_num(0.0)
        outs.append(p @ v)
        if scores is not None:
            scores[i, :, :n] += p.view(c["hkv"], group * nq, n).sum(1)
    o = torch.stack(outs)
    return o if scores is None else {"o": o, "scores": scores}
