"""Eviction from a K/V cache by accumulated attention weight.

A cache that is to stay within a budget keeps, per kv-head, its most recent keys and those that attention has given the
most weight so far.  Decode steps add each key's weight to its score as they attend, and every so often the cache is
cut down to the best:

    o, scores = attention_scored(q, k, v, scores=scores, causal=True, seqlens_k=lens)
    (k, v), scores, index, lens = evict_kv(scores, (k, v), keep, recent=recent, seqlens_k=lens)

Both take 16-bit caches and 4-bit ones (whose codes and pairs are four caches to ``evict_kv``).  The reference package
has neither.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _hip
from .int4 import attention_lengths_reference, dequantize_kv_int4
from .ops import _pick_backend


def attention_scored(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scores: Optional[torch.Tensor] = None,
                     causal: bool = False, scale: Optional[float] = None, seqlens_k: Optional[torch.Tensor] = None,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                     split_len: Optional[int] = None):
    """Attention that also scores the keys: (o [B, Hq, Nq, D], new scores fp32 [B, Hkv, Nk]) with

        new[b, h, j] = scores[b, h, j] + the attention weight of key j, summed over the q-heads of kv-head h and the
                       queries

    q [B, Hq, Nq, D] fp16/bf16, D in {64, 128, 256}; k, v [B or 1, Hkv, Nk, D] in q's type, or 4-bit codes with
    ``k_scale`` / ``v_scale`` (see ``attention_int4``).  ``scores`` (zeros if None) is not changed.  ``seqlens_k`` (int32
    [B]): the keys of each sequence; the rows behind them are not read and keep their scores.

    Made for decode steps, and for the last queries of a prompt: the scores of every (q-head, query, key) are held for
    the duration of the call, 4 bytes each."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if q.is_cuda and _pick_backend(q) == "hip":
        return _hip.cache_attention(q, k, v, k_scale, v_scale, causal, scale, split_len, seqlens_k=seqlens_k, scores=scores,
                                    return_scores=True)
    if _hip.check_cache_attention(q, k, v, k_scale, v_scale):
        k, v = dequantize_kv_int4(k, k_scale), dequantize_kv_int4(v, v_scale)
    if scores is not None:
        _hip.check_scores(scores, (q.shape[0], k.shape[1], k.shape[2]))
    if seqlens_k is not None:
        _hip.check_lengths(seqlens_k, q.shape[0])
    o, _, weights = attention_lengths_reference(q, k, v, causal, scale, seqlens_k, scored=True)
    return o, weights if scores is None else scores + weights


def evict_kv(scores: torch.Tensor, caches: Sequence[torch.Tensor], keep: int, recent: int = 0,
             seqlens_k: Optional[torch.Tensor] = None, out: Optional[Sequence[torch.Tensor]] = None):
    """Cut caches down to the ``keep`` keys that matter most, per sequence and kv-head.

    scores fp32 [B, Hkv, N]; caches: up to eight tensors [B, Hkv, N, ...] of any type (K, V, and for a 4-bit cache the
    pairs); ``seqlens_k`` int32 [B]: keys per sequence (default N).  A sequence with n > keep keys keeps its last
    ``recent`` ones and the keep - recent others of the highest scores (equal scores: the lower index; a NaN counts as
    the highest), in their order; one with n <= keep keeps all.  Returns

        caches   [B, Hkv, rows, ...], rows = min(keep, N), zeros past a sequence's keys
        scores   fp32 [B, Hkv, rows], zeros past them
        index    int32 [B, Hkv, rows], the keys' positions, -1 past them
        lengths  int32 [B], min(n, keep)

    ``out``: tensors [B, Hkv, >= rows, ...] to write the caches into (their further rows are left as they are); they
    must not share memory with the inputs."""
    caches = list(caches)
    out = None if out is None else list(out)
    keep, recent = int(keep), int(recent)
    if scores.is_cuda and _pick_backend(scores) == "hip":
        return _hip.evict_kv(scores, caches, keep, recent, seqlens_k, out)
    _hip.check_evict(scores, caches, keep, recent, seqlens_k, out)
    b, _, n = scores.shape
    keep, recent = min(keep, n), min(recent, n)
    end = torch.full((b,), n, dtype=torch.int32, device=scores.device) if seqlens_k is None else seqlens_k.clamp(0, n)
    end3 = end.long()[:, None, None]
    key = torch.arange(n, device=scores.device).expand(scores.shape)
    # by class (recent, other, no key), then by score, then by index
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices
    cls = torch.where(key >= end3, 2, torch.where(key >= end3 - recent, 0, 1))
    order = order.gather(-1, torch.sort(cls.gather(-1, order), dim=-1, stable=True).indices)
    index = torch.sort(order[..., :keep], dim=-1).values
    index = torch.where(index < end3, index, -1)

    def rows(t):
        at = index.clamp(min=0).view(*index.shape, *[1] * (t.dim() - 3)).expand(*index.shape, *t.shape[3:])
        keep_ = (index >= 0).view(*index.shape, *[1] * (t.dim() - 3))
        got = torch.gather(t, 2, at)
        return torch.where(keep_, got, torch.zeros_like(got))

    kept = [rows(t) for t in caches]
    if out is not None:
        for o, t in zip(out, kept):
            o[:, :, :keep] = t
        kept = out
    return kept, rows(scores), index.to(torch.int32), end.clamp(max=keep)
