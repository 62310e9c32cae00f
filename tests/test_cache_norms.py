"""The norm tolerance of cache_norms on the CPU: attention rounded as the kernels round passes it, planted mistakes do not."""
import math

import pytest
import torch

import fused_attn
from cache_norms import check_rows, deviation, row_errors
from oracle import cache_oracle as cor

N = 1000


def _inputs(dtype, d):
    g = torch.Generator().manual_seed(d)
    q = torch.randn(1, 8, 1, d, generator=g).to(dtype)
    size = torch.exp(0.5 * torch.randn(d, generator=g))
    kv = [fused_attn.quantize_kv_int4(torch.randn(1, 2, N, d, generator=g) * size) for _ in "kv"]
    return q, kv


def _rounded(q, k, v4, vs, terms, drop=None):
    """Attention in float64 but for P 16 scale, held in bf16 (the sum of ``terms`` of them), and the output.  ``drop``: the
    rows that V's product reads, in place of v4's."""
    group = q.shape[1] // k.shape[1]
    s = q.double() @ k.repeat_interleave(group, 1).transpose(-1, -2).contiguous() / math.sqrt(q.shape[-1])
    p = torch.exp(s - s.amax(-1, keepdim=True))
    c, sc, z = (x.repeat_interleave(group, 1) for x in
                (torch.stack([v4 & 15, v4 >> 4], -1).flatten(-2).double(), vs[..., 0].double(), vs[..., 1].double()))
    big = 16 * p * sc[:, :, None]
    held = torch.zeros_like(big)
    for _ in range(terms):
        held = held + (big - held).bfloat16().double()
    if drop is not None:
        c = drop(c)
    o = held @ (1 + c / 16) - (1 + 7.5 / 16) * held.sum(-1, keepdim=True) + (p * (z + 7.5 * sc)[:, :, None]).sum(-1, keepdim=True)
    return (o / p.sum(-1, keepdim=True)).to(q.dtype)


def _tile_of(at, other):
    def drop(c):
        c = c.clone()
        c[:, :, at:at + 32] = c[:, :, other:other + 32] if other is not None else 0
        return c
    return drop


def _tail(c):
    c = c.clone()
    c[:, :, -8:] = 0
    return c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_norm_tolerance_tells_mistakes_from_roundings(dtype, d):
    q, ((k4, ks), (v4, vs)) = _inputs(dtype, d)
    k, v, dev = cor.values(k4, ks), cor.values(v4, vs), deviation(v4, vs)
    terms = 2 if dtype == torch.float16 else 1
    check_rows(_rounded(q, k, v4, vs, terms), q, k, v, dev)
    for drop in (_tile_of(320, None), _tile_of(320, 192), _tail):  # a tile of zeros, the wave's previous tile, the last rows
        err, tol = row_errors(_rounded(q, k, v4, vs, terms, drop), q, k, v, dev)
        assert (err > tol).all(), (err / tol).min()
    if dtype == torch.float16:  # P in one bf16 term
        err, tol = row_errors(_rounded(q, k, v4, vs, 1), q, k, v, dev)
        assert (err > tol).all(), (err / tol).min()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norm_tolerance_of_16_bit_rows(dtype):
    q, kv = _inputs(dtype, 128)
    k, v = (cor.values(*x).to(dtype) for x in kv)
    s = q.double() @ k.double().repeat_interleave(4, 1).transpose(-1, -2).contiguous() / math.sqrt(128)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    vv = v.double().repeat_interleave(4, 1)
    got = ((p.to(dtype).double() @ vv) / p.sum(-1, keepdim=True)).to(dtype)
    check_rows(got, q, k.double(), v.double())
    for drop in (_tile_of(320, None), _tile_of(320, 192), _tail):
        got = ((p.to(dtype).double() @ drop(vv)) / p.sum(-1, keepdim=True)).to(dtype)
        err, tol = row_errors(got, q, k.double(), v.double())
        assert (err > tol).all(), (err / tol).min()
