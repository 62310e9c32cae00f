"""Pages of a K/V cache: block tables and slots built on the GPU from request lengths.

A serving step takes pages for its new tokens, writes their keys and values, and attends:

    slots, cu_seqlens, seqlens_k, num_free = allocate_pages(block_table, seqlens_k, new_lens, free_pages, num_free,
                                                            page_size, num_tokens)
    append_kv_paged(k, v, k_cache, v_cache, slots)               # k, v packed [num_tokens, Hkv, D]
    o = attention_paged(q, k_cache, v_cache, block_table, seqlens_k, causal=True, max_seqlen_k=...)
    seqlens_k, num_free = release_pages(block_table, seqlens_k, done, free_pages, num_free, page_size)

The lengths, the table and the list of free pages stay on the device: nothing waits for it, and a step can be captured
into a graph.  ``free_pages`` int32 [F] is a stack, whose first ``num_free`` entries (int32, one element) are the pages
nobody holds.  Request b's keys fill the pages of its row of ``block_table`` in order; requests may share whole pages at
the start of their rows (see ``attention_shared_prefix``).

On the GPU each function is one HIP kernel; CPU tensors, or ``FUSED_ATTN_BACKEND=reference``, take the torch form.  The
reference package has no paged cache.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _hip
from .ops import _pick_backend


def allocate_pages(block_table: torch.Tensor, seqlens_k: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
                   num_free: torch.Tensor, page_size: int, num_tokens: int):
    """Pages and slots for ``new_lens[b]`` (int32 [B]; 0 or less: none) new tokens of every request b, which holds
    ``seqlens_k[b]`` (int32 [B]) keys.  The tokens are packed, ``num_tokens`` of them.  Returns

        slots       int64 [num_tokens]: page * page_size + offset of every token, -1 where it has none
        cu_seqlens  int32 [B + 1]: where each request's tokens start (as ``attention_varlen`` takes it)
        seqlens     int32 [B]: keys per request with the new ones
        num_free    int32, of num_free's shape: free pages left

    and writes the new pages into the rows of ``block_table`` (int32 [B, columns]).  Pages are taken from the end of
    ``free_pages``, requests in order.  A request gets all its tokens or none: one whose keys would pass its row's
    columns, whose tokens would pass num_tokens, or that needs pages when too few are left for it and those before it,
    keeps its length and its row, and its tokens have slot -1."""
    args = (block_table, seqlens_k, new_lens, free_pages, num_free, int(page_size), int(num_tokens))
    out = None if _hip.native is None else _hip.native.allocate_pages(*args)
    if out is not None:
        return out
    if block_table.is_cuda and _pick_backend(block_table) == "hip":
        return _hip.allocate_pages(*args)
    _hip.check_pages(block_table, seqlens_k, free_pages, num_free, args[5], new_lens=new_lens, num_tokens=args[6])
    page, tokens, cols, dev = args[5], args[6], block_table.shape[1], block_table.device
    n, m = seqlens_k.long().clamp(min=0), new_lens.long().clamp(min=0)
    free = num_free.reshape(()).long().clamp(0, free_pages.numel())
    end = torch.cumsum(m, 0)
    have, want = -(-n // page), -(-(n + m) // page)
    fits = (n + m <= min(cols * page, 2 ** 31 - 1)) & (end <= tokens)
    need = torch.where(fits, want - have, 0)
    ok = fits & ((need == 0) | (torch.cumsum(need, 0) <= free))
    need = torch.where(ok, need, 0)
    first = torch.cumsum(need, 0) - need
    seq, j = _ragged(need)
    block_table[seq, have[seq] + j] = free_pages[free - 1 - first[seq] - j]
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=dev)
    seq, j = _ragged(torch.where(ok, m, 0))
    pos = n[seq] + j
    entry = block_table[seq, pos // page].long()
    slots[(end - m)[seq] + j] = torch.where(entry >= 0, entry * page + pos % page, -1)
    cu = torch.zeros(n.numel() + 1, dtype=torch.int32, device=dev)
    cu[1:] = end.clamp(max=tokens)
    return slots, cu, torch.where(ok, n + m, n).to(torch.int32), (free - need.sum()).to(torch.int32).reshape(num_free.shape)


def _ragged(counts: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(i, j) for every i and 0 <= j < counts[i]."""
    i = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    return i, torch.arange(i.numel(), device=counts.device) - (torch.cumsum(counts, 0) - counts)[i]


def release_pages(block_table: torch.Tensor, seqlens_k: torch.Tensor, done: torch.Tensor, free_pages: torch.Tensor,
                  num_free: torch.Tensor, page_size: int, keep_lens: Optional[torch.Tensor] = None):
    """Requests with ``done[b]`` (bool or uint8 [B]) give their pages back: they are put on the end of ``free_pages`` in
    place, requests in order, their pages in order.  Returns (seqlens int32 [B]: 0 for those, num_free: free pages now).

    ``keep_lens`` (int32 [B]): keys at the start of a request that others share; the whole pages they fill stay out of
    the list.  A request whose pages the list has no room for keeps them and its length.  ``block_table`` is not changed:
    a row's entries past its length mean nothing.  What a row holds is put back as it is: a negative entry too (tokens that
    get it later have slot -1), and a page that two finished requests share twice, unless keep_lens leaves it out."""
    args = (block_table, seqlens_k, done, free_pages, num_free, int(page_size), keep_lens)
    out = None if _hip.native is None else _hip.native.release_pages(*args[:5], keep_lens, args[5])
    if out is not None:
        return out
    if block_table.is_cuda and _pick_backend(block_table) == "hip":
        return _hip.release_pages(*args)
    _hip.check_pages(block_table, seqlens_k, free_pages, num_free, args[5], done=done, keep_lens=keep_lens)
    page, cols = args[5], block_table.shape[1]
    n = seqlens_k.long().clamp(min=0)
    free = num_free.reshape(()).long().clamp(0, free_pages.numel())
    keep = torch.zeros_like(n) if keep_lens is None else keep_lens.long().clamp(min=0) // page
    count = torch.where(done.bool(), ((-(-n // page)).clamp(max=cols) - keep).clamp(min=0), 0)
    ok = done.bool() & ((count == 0) | (torch.cumsum(count, 0) + free <= free_pages.numel()))
    count = torch.where(ok, count, 0)
    seq, j = _ragged(count)
    free_pages[free + torch.arange(seq.numel(), device=n.device)] = block_table[seq, keep[seq] + j]
    return torch.where(ok, 0, n).to(torch.int32), (free + count.sum()).to(torch.int32).reshape(num_free.shape)


def append_kv_paged(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    slots: torch.Tensor) -> None:
    """Write packed rows k, v [T, Hkv, D] at ``slots`` (int64 [T], as ``allocate_pages`` gives them) of 16-bit pools
    k_cache, v_cache [num_pages, Hkv, page_size, D] of the same type, in place; any strides with unit D stride, D a
    multiple of 8.  A token with a slot outside [0, num_pages * page_size) is not written; no two may have the same one.

    (An FP8 pool shares a scale among 64 keys and cannot take single rows; 4-bit pools have ``append_kv_int4``.)"""
    if _hip.native is not None and _hip.native.append_kv_paged(k, v, k_cache, v_cache, slots):
        return
    if k.is_cuda and _pick_backend(k) == "hip":
        return _hip.append_kv_paged(k, v, k_cache, v_cache, slots)
    _hip.check_append_paged(k, v, k_cache, v_cache, slots)
    page = k_cache.shape[2]
    keep = (slots >= 0) & (slots < k_cache.shape[0] * page)
    at = slots[keep]
    k_cache[at // page, :, at % page] = k[keep]
    v_cache[at // page, :, at % page] = v[keep]
