"""4-bit K/V cache: a quarter of a 16-bit cache's bytes, which are what decode waits for.

A row (one token of one kv-head) is held as 4-bit codes between its own ends, with an fp16 pair a row:

    zero = fp16(min), scale = fp16((max - min) / 15), code = clamp(round((x - zero) / scale), 0, 15)
    value = code * scale + zero

    k4, ks = quantize_kv_int4(k)          # uint8 [B, Hkv, N, D/2] (even channels in the low halves), fp16 [B, Hkv, N, 2]
    v4, vs = quantize_kv_int4(v)
    o = attention_int4(q, k4, ks, v4, vs, causal=True)

The pair belongs to the row, so that rows are appended one token at a time (``append_kv_int4``, dense or paged), and
picked one at a time (``evict_kv``); the FP8 cache shares a scale among 64 keys and allows neither without re-coding.
The minimum and maximum are held to +-65504; an infinity counts as the row's end, a NaN makes its row's pair NaN.

On the GPU these are HIP kernels for D in {64, 128, 256}; the writer, the reader and, at multiples of 8, ``append_kv_int4``
take the torch form at other D, and every function does for CPU tensors or ``FUSED_ATTN_BACKEND=reference``.  The reference package has no 4-bit cache.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _hip
from .ops import _pick_backend
from .reference import attention_reference, causal_mask, lse_reference

FP16_MAX = 65504.0


def quantize_kv_int4(x: torch.Tensor, out: Optional[tuple] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [B, Hkv, N, D] (fp32/fp16/bf16, any strides) -> (codes uint8 [B, Hkv, N, D/2], pairs fp16 [B, Hkv, N, 2]).

    ``out`` = (codes, pairs) to write into, views of a larger cache among them (``cache[:, :, n0:n1]``)."""
    if x.dim() != 4 or x.shape[-1] % 2 or not x.is_floating_point():
        raise RuntimeError(f"x must be floating [B, Hkv, N, D] with an even D, got {x.dtype} {tuple(x.shape)}")
    if x.is_cuda and _pick_backend(x) == "hip" and x.shape[-1] in _hip.INT4_HEAD_DIMS:
        return _hip.quantize_kv_int4(x, out)
    codes, scale = _quantize_kv_int4_torch(x)
    if out is None:
        return codes, scale
    _hip.check_int4_rows(*out, "out", codes.shape)
    out[0].copy_(codes)
    out[1].copy_(scale)
    return tuple(out)


def _quantize_kv_int4_torch(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    x = x.float()
    lo, hi = (t.clamp(-FP16_MAX, FP16_MAX) for t in (x.amin(-1), x.amax(-1)))
    zero, scale = lo.half(), ((hi - lo) * (1.0 / 15.0)).half()
    step = scale.float()[..., None]
    code = torch.round((x - zero.float()[..., None]) / step)
    code = torch.where(step > 0, code, torch.zeros_like(code)).clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([scale, zero], -1)


def dequantize_kv_int4(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """What 4-bit rows stand for, [B, Hkv, N, D]: code * scale + zero in fp32, rounded to ``dtype``.  (Prefill-sized
    calls over a 4-bit cache: read it back once and call ``attention``.)"""
    _hip.check_int4_rows(codes, scale, "codes")
    if codes.is_cuda and _pick_backend(codes) == "hip" and 2 * codes.shape[-1] in _hip.INT4_HEAD_DIMS \
            and dtype in (torch.float32, torch.float16, torch.bfloat16):
        return _hip.dequantize_kv_int4(codes, scale, dtype)
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return (code.float() * scale[..., :1].float() + scale[..., 1:].float()).to(dtype)


def append_kv_int4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_cache: torch.Tensor, v_scale: torch.Tensor, seqlens_k: torch.Tensor,
                   block_table: Optional[torch.Tensor] = None) -> None:
    """Write new tokens k, v [B, Hkv, n, D] into a 4-bit cache in place (one launch; the torch form waits for the device).

    Token i of sequence b goes to position ``seqlens_k[b] + i`` (int32 [B], the keys it holds before the call, which
    the call leaves as they are) of k_cache / v_cache uint8 [B, Hkv, capacity, D/2], or with ``block_table`` (int32
    [B, pages]) of pools [num_pages, Hkv, page_size, D/2]; k_scale / v_scale are their pairs [..., 2].  A token past
    the cache's end, or whose page is outside the pool, is not written.  No two sequences may share a written page."""
    args = (k, v, k_cache, k_scale, v_cache, v_scale, seqlens_k, block_table)
    if k.is_cuda and _pick_backend(k) == "hip" and k.dim() == 4 and k.shape[-1] in _hip.INT4_HEAD_DIMS:
        return _hip.append_kv_int4(*args)
    _hip.check_append(*args)
    b, _, n, _ = k.shape
    page = k_cache.shape[2]
    cap = page if block_table is None else block_table.shape[1] * page
    pos = seqlens_k.long()[:, None] + torch.arange(n, device=k.device)
    seq, token = ((pos >= 0) & (pos < cap)).nonzero(as_tuple=True)
    at, pos = seq, pos[seq, token]
    if block_table is not None:
        at, pos = block_table[seq, pos // page].long(), pos % page
        ok = (at >= 0) & (at < k_cache.shape[0])
        seq, token, at, pos = (t[ok] for t in (seq, token, at, pos))
    for x, codes, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        c, s = _quantize_kv_int4_torch(x)
        codes[at, :, pos], scale[at, :, pos] = c[seq, :, token], s[seq, :, token]


def _weights_reference(q, k, causal: bool, scale: float) -> torch.Tensor:
    """The probabilities of ``attention_reference`` [B, Hkv, Nk], summed over a kv-head's q-heads and the queries."""
    b, hq, nq, d = q.shape
    hkv, nk = k.shape[1], k.shape[2]
    s = torch.matmul(q.float().reshape(b, hkv, hq // hkv * nq, d), k.float().transpose(-1, -2)) * scale
    if causal:
        s = s.masked_fill(~causal_mask(nq, nk, device=q.device).repeat(hq // hkv, 1), -math.inf)
    return torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0).sum(2)  # (rows without a visible key: NaN)


def attention_lengths_reference(q, k, v, causal: bool, scale: float, seqlens_k=None, scored: bool = False):
    """The unfused path over the first ``seqlens_k[b]`` keys of each sequence: (o, lse, and if ``scored`` the weights
    [B, Hkv, Nk])."""
    b, hq, nq, _ = q.shape
    hkv, nk = k.shape[1], k.shape[2]
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    weights = torch.zeros(b, hkv, nk, dtype=torch.float32, device=q.device) if scored else None
    lens = [nk] * b if seqlens_k is None else [min(max(n, 0), nk) for n in seqlens_k.tolist()]
    for i, n in enumerate(lens):
        at = i if k.shape[0] == b else 0
        ki, vi, qi = k[at:at + 1, :, :n], v[at:at + 1, :, :n], q[i:i + 1]
        o[i:i + 1] = attention_reference(qi, ki, vi, causal=causal, scale=scale)
        lse[i:i + 1] = lse_reference(qi, ki, causal=causal, scale=scale)
        if scored:
            weights[i, :, :n] = _weights_reference(qi, ki, causal, scale)[0]
    return o, lse, weights


def attention_int4(q: torch.Tensor, k4: torch.Tensor, k_scale: torch.Tensor, v4: torch.Tensor, v_scale: torch.Tensor,
                   causal: bool = False, scale: Optional[float] = None, seqlens_k: Optional[torch.Tensor] = None,
                   split_len: Optional[int] = None, return_lse: bool = False):
    """Attention of q [B, Hq, Nq, D] (fp16/bf16) over a 4-bit cache: k4, v4 uint8 [B or 1, Hkv, Nk, D/2] with pairs fp16
    [B or 1, Hkv, Nk, 2].  Returns [B, Hq, Nq, D] in q's type, and with ``return_lse`` the natural-log LSE
    (fp32 [B, Hq, Nq], -inf for rows without keys).

    ``seqlens_k`` (int32 [B], on the device): only the first seqlens_k[b] rows of sequence b are keys, and ``causal``
    aligns its queries to their end; the rows behind them are not read.  Any number of queries is accepted; the kernel
    is made for decode.  From about 64 (one sequence) to 128 queries (eight; 32 q-heads over 8, 8192 keys, D <= 128; twice
    that at D=256) ``dequantize_kv_int4`` and ``attention`` are faster together: 8 x 128 queries of D=128 in 208 us, 271
    here, 16 queries in 144 and 72."""
    if k4.dtype != torch.uint8:
        raise RuntimeError(f"attention_int4 needs 4-bit K/V (uint8), got {k4.dtype}")
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if not q.is_cuda or _pick_backend(q) != "hip":
        _hip.check_cache_attention(q, k4, v4, k_scale, v_scale)
        if seqlens_k is not None:
            _hip.check_lengths(seqlens_k, q.shape[0])
        k, v = dequantize_kv_int4(k4, k_scale), dequantize_kv_int4(v4, v_scale)
        o, lse, _ = attention_lengths_reference(q, k, v, causal, scale, seqlens_k)
        return (o, lse) if return_lse else o
    return _hip.cache_attention(q, k4, v4, k_scale, v_scale, causal, scale, split_len, seqlens_k=seqlens_k,
                                return_lse=return_lse)
