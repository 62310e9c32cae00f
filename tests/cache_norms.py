"""A tolerance on the norm of each output row of attention over a cache, beside the elementwise one of cache_helpers.

The elementwise bound counts every rounding at its worst and grows with the channels and keys; roundings are independent of
each other, and the norm of a row's error follows their mean square.  With p the weights (float64), u = half a step of the
output's type and uP that of the type in which P meets V,

    |got - o| <= u |o|                                       the output's own rounding
               + 2 uP sqrt(sum_d sum_j p_j^2 dev_jd^2)       P's: each of at most uP p_j, mean square at most a third of it
               + 2^-13 (sqrt(sum_d sum_j p_j^2 v_jd^2) + |o|)  the scores', see below

dev: what P's rounding meets: V itself (16 bits, uP of q's type), or its deviation from the middle of its row, scale
(code - 7.5) (4 bits; P is bf16, 2^-8, and for fp16 outputs two bf16 terms, 2^-16).  The scores: sums of D products in fp32,
at 4 bits of q (1 + code/16), whose partial sums stay below 256 here (D <= 256, |q| about 1): each of the D additions is off
by at most 2^-24 * 256, together sqrt(D) of that, 2^-12, times 16 scale c < 0.4 = 16 * 0.4 / sqrt(256): 2^-13.3; the sums of
16-bit products are smaller."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def deviation(codes, pairs):
    """scale (code - 7.5) of 4-bit rows, float64."""
    c = codes.to(torch.int64)
    both = torch.stack([c % 16, c // 16], -1).flatten(-2).double()
    return (both - 7.5) * pairs[..., 0:1].double()


def row_errors(got, q, k, v, dev=None, causal=False, lens=None):
    """(error norms, their tolerances) of the output rows [B, Hq, Nq]; k, v float64 values [B or 1, Hkv, N, D], ``dev`` what
    P's rounding meets (None: 16-bit V).  Rows behind lens[b] are left out, whatever they hold."""
    b, hq, nq, d = q.shape
    up = U[q.dtype] if dev is None else (2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -16)
    err, tol = (torch.zeros(b, hq, nq, dtype=torch.float64, device=q.device) for _ in range(2))
    for i in range(b):
        n = k.shape[2] if lens is None else min(max(int(lens[i]), 0), k.shape[2])
        at = i if k.shape[0] == b else 0
        for h in range(hq):
            kh = h // (hq // k.shape[1])
            kk, vv = k[at, kh, :n], v[at, kh, :n]
            s = (q[i, h].double() @ kk.t().contiguous()) / math.sqrt(d)
            if causal:
                row = torch.arange(nq, device=q.device)[:, None]
                s = s.masked_fill(torch.arange(n, device=q.device)[None] > row + n - nq, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            o = p @ vv
            size, noise = o.norm(dim=-1), ((p * p) @ (vv * vv)).sum(-1).sqrt()
            met = noise if dev is None else ((p * p) @ dev[at, kh, :n].square()).sum(-1).sqrt()
            err[i, h] = (got[i, h].double() - o).norm(dim=-1)
            tol[i, h] = U[q.dtype] * size + 2 * up * met + 2.0 ** -13 * (noise + size)
    return err, tol


def check_rows(got, *args, **kw):
    assert torch.isfinite(got).all()
    err, tol = row_errors(got, *args, **kw)
    worst = (err / tol.clamp(min=1e-30)).max()
    assert (err <= tol).all(), f"a row's error is {worst:.2f} times its tolerance"
    return float(worst)
