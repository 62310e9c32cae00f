"""Inputs and tolerances shared by the GPU tests of the 4-bit cache and of scored attention."""
import math

import torch

import fused_attn
from oracle import cache_oracle as cor

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(shape, dtype, seed=0):
    """Rows whose channels differ in size and offset."""
    g = gen(seed)
    size = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=g))
    shift = 0.5 * torch.randn(shape[-1], device="cuda", generator=g)
    return (torch.randn(shape, device="cuda", generator=g) * size + shift).to(dtype)


def cache(b, hkv, n, d, seed=0):
    """A 4-bit cache made by the torch form (on the CPU), so that attention is tested apart from the GPU's writer."""
    codes, pairs = fused_attn.quantize_kv_int4(rows((b, hkv, n, d), torch.float32, seed).cpu())
    return codes.cuda(), pairs.cuda()


def score_error(q, k, pairs, scale):
    """Bound on the error of a score (natural log units): a dot product of D products summed in fp32 in any order is off
    by at most D half-steps of the sum of their sizes, and a few more roundings follow.  4 bits: the product's second
    factor is 1 + code/16 (below 2) times 16 * scale, and zero times sum(q) is added."""
    d = q.shape[-1]
    size = q.double().abs().sum(-1).amax() * (k.double().abs().amax() if pairs is None else
                                               (32 * pairs[..., 0].double() + pairs[..., 1].double().abs()).nan_to_num().amax())
    return float((d + 8) * U[torch.float32] * abs(scale) * size)


def check(got, o, lse, w, q, k, v, pairs=None, scale=None, got_lse=None, got_w=None, before=None):
    """Outputs against the oracle's (float64).  ``pairs``: those of K and V for a 4-bit cache (k, v its values).

    o: its own rounding (half a step), the weights' error, and P's rounding, which meets the deviation of a 4-bit value
    from the middle of its row (7.5 scale at most; bf16), or a 16-bit value (q's type).  Sums in fp32 add less than
    2^-16 of the largest value."""
    assert got.shape == q.shape and got.dtype == q.dtype
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if k.shape[2] == 0:
        assert (got == 0).all()
        return
    delta = 2 * score_error(q, k, None if pairs is None else pairs[0], scale) + 2.0 ** -20  # a weight's relative error
    vmax = float(v.nan_to_num().abs().amax())
    p_err = U[q.dtype] * vmax if pairs is None else U[torch.bfloat16] * 7.5 * float(pairs[1][..., 0].double().nan_to_num().amax())
    tol = U[q.dtype] * o.abs() + p_err + (delta + 2.0 ** -16) * vmax
    err = (got.double() - o).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), f"o off by {(err - tol).max():.3e} over the tolerance"
    if got_lse is not None:
        assert torch.equal(torch.isneginf(got_lse), torch.isneginf(lse))
        fine = ~torch.isneginf(lse)
        off = (got_lse.double() - lse)[fine].abs()
        assert (off <= delta + 2.0 ** -20 * (1 + lse[fine].abs())).all(), f"lse off by {off.max():.3e}"
    if got_w is not None:
        base = torch.zeros_like(w) if before is None else before.double()
        off = (got_w.double() - base - w).abs()
        # the weights' relative error, the sum over rows, and the addition to what was there
        rows_ = q.shape[1] // k.shape[1] * q.shape[2]
        tol = w * (delta + rows_ * U[torch.float32]) + U[torch.float32] * (base + w) * 2 + 1e-30
        assert (off <= tol).all(), f"scores off by {(off - tol).max():.3e} over the tolerance"


def garbage_behind(codes, pairs, lens):
    """NaN pairs (or rows) behind each sequence's keys: nothing may read them."""
    for i, n in enumerate(lens):
        n = min(max(n, 0), codes.shape[2])
        if pairs is None:
            codes[i, :, n:] = math.nan
        else:
            codes[i, :, n:] = 255
            pairs[i, :, n:] = math.nan


oracle = cor
