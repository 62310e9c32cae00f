"""Decode attention for requests that share the start of their context.

Requests behind one system prompt, or parallel answers to one document, hold the same pages at the start of their
block-table rows.  ``attention_paged`` reads those keys once per request; here a group's rows (requests x q-heads of a
kv-head x queries) meet them together, as the rows of one matrix product, and each request's own keys behind them as in
``attention_paged``.  Both parts' partials are merged by their log-sum-exps, so the result is that of

    attention_paged(q, k_cache, v_cache, block_table, seqlens_k, ...)

up to the rounding of another order of sums.  The reference package has no paged cache.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _hip
from .ops import _pick_backend
from .paged import attention_paged


def attention_shared_prefix(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                            seqlens_k: torch.Tensor, prefix_lens: Union[int, torch.Tensor],
                            cu_groups: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                            max_prefix_len: Optional[int] = None, max_suffix_len: Optional[int] = None,
                            split_len: Optional[int] = None, return_lse: bool = False,
                            k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
    """Attention of q [B, Hq, Nq, D] (fp16/bf16, D in {64, 128, 256}) over a paged cache, 16-bit or FP8, whose requests
    share prefixes.  ``block_table``, ``seqlens_k`` (all keys of a request, the shared ones among them), ``causal``,
    ``scale``, ``return_lse`` and the FP8 pools' ``k_scale`` / ``v_scale`` are those of ``attention_paged``.

    Group g is the requests ``cu_groups[g]`` to ``cu_groups[g + 1] - 1`` (int32 [G + 1] from 0 to B; None: one group, the
    whole batch), whose rows name the same keys in their first ``prefix_lens[g]`` positions (int32 [G], or one number for
    every group); the pages may be the same or copies (of an FP8 page: with its scales).  A prefix may be 0, need not fill
    whole pages, and a request may be shorter than it (a padded batch's empty ones among them).  The shared keys are read
    through the row of a request that holds them all, and at most as far as the longest request of the group has them.
    (On the GPU a shared 64-key block of FP8 V whose scale is 0, or below 2^-90 of another's in its partition, counts as
    zeros, and an infinite or NaN scale makes NaN of the rows that see the block.)

    ``max_prefix_len`` and ``max_suffix_len`` size the grid: the largest of prefix_lens, and of a request's keys behind
    its group's prefix.  When omitted they are read from the device, which waits for it; as numbers, they let the call be
    captured into a graph.  Longer prefixes than max_prefix_len are shared up to it, the rest of them counts as own
    keys; a request with more than max_suffix_len keys of its own counts as one that ends there (its causal queries too).
    ``split_len``: keys per partition, a multiple of 64 that spans at most 128 pages (of FP8 pools: at most 4096 keys).  All
    three are at most 2^29."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    number = not isinstance(prefix_lens, torch.Tensor)
    if _hip.native is not None and max_suffix_len is not None and not return_lse and split_len is None \
            and (number or max_prefix_len is not None):
        bound = prefix_lens if max_prefix_len is None else min(max_prefix_len, prefix_lens) if number else max_prefix_len
        o = _hip.native.shared_prefix(q, k_cache, v_cache, block_table, seqlens_k, None if number else prefix_lens, cu_groups,
                                      k_scale, v_scale, max(0, int(bound)), max(0, int(max_suffix_len)), bool(causal), float(scale), 0)
        if o is not None:
            return o
    _hip.check_shared_prefix(q, k_cache, v_cache, block_table, seqlens_k, prefix_lens, cu_groups)
    longest = [int(n) for n in (max_prefix_len, prefix_lens if number else None) if n is not None]
    _hip.check_shared_bounds(max_prefix_len=min(longest) if longest else None, max_suffix_len=max_suffix_len, split_len=split_len)
    if not q.is_cuda or _pick_backend(q) != "hip":
        if max_suffix_len is not None:
            end = _prefixes(seqlens_k, prefix_lens, cu_groups, max_prefix_len) + max(0, int(max_suffix_len))
            seqlens_k = torch.minimum(seqlens_k.long(), end).to(torch.int32)
        return attention_paged(q, k_cache, v_cache, block_table, seqlens_k, causal=causal, scale=scale, return_lse=return_lse,
                               k_scale=k_scale, v_scale=v_scale)
    if max_prefix_len is None:
        max_prefix_len = prefix_lens if number else int(prefix_lens.max().item()) if prefix_lens.numel() else 0
    if max_suffix_len is None:
        max_suffix_len = _longest_suffix(seqlens_k, prefix_lens, cu_groups, max_prefix_len)
    if number:  # (the kernels hold every group's prefix to max_prefix_len)
        max_prefix_len, prefix_lens = min(int(max_prefix_len), int(prefix_lens)), None
    return _hip.shared_prefix(q, k_cache, v_cache, block_table, seqlens_k, prefix_lens, cu_groups, max(0, int(max_prefix_len)),
                              max(0, int(max_suffix_len)), causal=causal, scale=scale, split_len=split_len,
                              return_lse=return_lse, k_scale=k_scale, v_scale=v_scale)


def _prefixes(seqlens_k: torch.Tensor, prefix_lens, cu_groups: Optional[torch.Tensor],
              max_prefix_len: Optional[int]) -> torch.Tensor:
    """The prefix of every request (int64 [B]), at most max_prefix_len; 0 for one of no group."""
    b, dev = seqlens_k.numel(), seqlens_k.device
    groups = 1 if cu_groups is None else cu_groups.numel() - 1
    p = prefix_lens.long() if isinstance(prefix_lens, torch.Tensor) else torch.full((groups,), int(prefix_lens), device=dev)
    p = p.clamp(min=0, max=None if max_prefix_len is None else max(0, int(max_prefix_len)))
    if cu_groups is None:
        return p.expand(b)
    request = torch.arange(b, device=dev)
    group = torch.searchsorted(cu_groups[1:].long().contiguous(), request, right=True)
    return torch.where((request >= cu_groups[0]) & (group < groups), p[group.clamp(max=groups - 1)], 0)


def _longest_suffix(seqlens_k: torch.Tensor, prefix_lens, cu_groups: Optional[torch.Tensor], max_prefix_len: int) -> int:
    """The most keys that a request has behind what its group shares (at most max_prefix_len)."""
    if seqlens_k.numel() == 0:
        return 0
    return max(0, int((seqlens_k.long() - _prefixes(seqlens_k, prefix_lens, cu_groups, max_prefix_len)).max().item()))
