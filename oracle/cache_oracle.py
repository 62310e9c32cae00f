"""ORACLE for the 4-bit cache, scored attention and eviction — test infrastructure, not product code.

Float64 (numpy for the rows and the eviction, torch for the products), from the definitions:

    zero = fp16(lo), scale = fp16((hi - lo) * fp32(1/15)), code = clamp(rint((x - zero) / scale), 0, 15)
    value = code * scale + zero

It is pinned by tests/test_cache_oracle.py: closed forms, the existing attention oracle and brute force.
"""
from __future__ import annotations

import math

import numpy as np
import torch

F16_MAX = np.float32(65504.0)


def encode(x: torch.Tensor):
    """(codes [..., D] 0..15, scale, zero as float16 [...]) of x [..., D], in the definition's fp32 steps."""
    x32 = x.detach().cpu().float().numpy()
    lo, hi = x32.min(-1), x32.max(-1)  # numpy's min and max keep NaN
    lo, hi = np.clip(lo, -F16_MAX, F16_MAX), np.clip(hi, -F16_MAX, F16_MAX)
    with np.errstate(all="ignore"):
        zero = lo.astype(np.float16)
        scale = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
        q = (x32 - zero.astype(np.float32)[..., None]) / scale.astype(np.float32)[..., None]
        code = np.clip(np.rint(q), 0, 15)
        code = np.where(scale.astype(np.float32)[..., None] > 0, code, 0).astype(np.uint8)
    return code, scale, zero


def pack(code: np.ndarray) -> np.ndarray:
    return code[..., 0::2] | (code[..., 1::2] << 4)


def values(codes: torch.Tensor, pairs: torch.Tensor) -> torch.Tensor:
    """What packed rows stand for, float64 on the codes' device."""
    c = codes.to(torch.int64)
    both = torch.stack([c % 16, c // 16], -1).flatten(-2).double()
    return both * pairs[..., 0:1].double() + pairs[..., 1:2].double()


def attention(q, k, v, causal=False, scale=None, lens=None):
    """(o, lse, weights) in float64 for q [B, Hq, Nq, D] and the first lens[b] rows of k, v [B or 1, Hkv, N, D];
    weights [B, Hkv, N] are the probabilities summed over the group's heads and the queries."""
    b, hq, nq, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    o = torch.zeros(b, hq, nq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq, nq), -math.inf, dtype=torch.float64, device=q.device)
    weights = torch.zeros(b, hkv, n, dtype=torch.float64, device=q.device)
    for i in range(b):
        m = n if lens is None else min(max(int(lens[i]), 0), n)
        if m == 0:
            continue
        at = i if k.shape[0] == b else 0
        for h in range(hq):
            kh = k[at, h // (hq // hkv), :m].double()
            s = (q[i, h].double() @ kh.t().contiguous()) * scale
            if causal:
                row = torch.arange(nq, device=q.device)[:, None]
                s = s.masked_fill(torch.arange(m, device=q.device)[None] > row + m - nq, -math.inf)
            lse[i, h] = torch.logsumexp(s, -1)
            p = torch.where(torch.isneginf(lse[i, h])[:, None], 0.0, torch.exp(s - lse[i, h][:, None]))
            o[i, h] = p @ v[at, h // (hq // hkv), :m].double()
            weights[i, h // (hq // hkv), :m] += p.sum(0)
    return o, lse, weights


def kept(scores: np.ndarray, n: int, keep: int, recent: int) -> list[int]:
    """Positions that stay of one head's scores: sorted by hand, NaN above every number, then the lower index."""
    n = min(max(n, 0), len(scores))
    if n <= keep:
        return list(range(n))
    old = n - recent
    rank = sorted(range(old), key=lambda j: (not np.isnan(scores[j]), 0.0 if np.isnan(scores[j]) else -float(scores[j]), j))
    return sorted(rank[:keep - recent] + list(range(old, n)))
