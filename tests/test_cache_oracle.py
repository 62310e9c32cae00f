"""The float64 oracle of the 4-bit cache and of eviction, pinned by closed forms, the attention oracle and brute force."""
import math

import numpy as np
import pytest
import torch

from oracle import attention_oracle as orc
from oracle import cache_oracle as cor


def test_codes_of_a_ramp_are_its_steps():
    x = torch.arange(16.0).repeat(4)[None] * 0.5 - 3.0  # scale 0.5 and zero -3 are exact
    code, scale, zero = cor.encode(x)
    assert scale[0] == 0.5 and zero[0] == -3.0
    assert np.array_equal(code[0], np.tile(np.arange(16), 4))


def test_halves_round_to_even_and_constant_rows_are_their_zero():
    x = torch.tensor([[0.0, 15.0, 0.5, 1.5, 2.5, 14.5]])
    assert cor.encode(x)[0].tolist() == [[0, 15, 0, 2, 2, 14]]
    code, scale, zero = cor.encode(torch.full((1, 8), 1.25))
    assert code.max() == 0 and scale[0] == 0 and zero[0] == 1.25


def test_a_value_is_within_half_a_step():
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(0))
    code, scale, zero = cor.encode(x)
    pairs = torch.from_numpy(np.stack([scale, zero], -1))
    y = cor.values(torch.from_numpy(cor.pack(code)), pairs)
    # half a step, and what rounding the ends to fp16 (2^-11 of each) leaves outside the 16 levels
    ends = x.abs().amax(-1, keepdim=True).double()
    tol = pairs[:, :1].double() * 0.5 + 2 * ends * 2.0 ** -11 + 15 * pairs[:, :1].double() * 2.0 ** -11
    assert ((y - x.double()).abs() <= tol).all()


def test_pack_puts_even_channels_low():
    assert cor.pack(np.array([[1, 2, 3, 15]], dtype=np.uint8)).tolist() == [[0x21, 0xf3]]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,n", [(1, 7), (5, 5), (3, 9), (9, 4)])
def test_attention_matches_the_attention_oracle(nq, n, causal):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, m, 32, generator=g) for h, m in ((4, nq), (2, n), (2, n)))
    o, lse, w = cor.attention(q, k, v, causal)
    torch.testing.assert_close(o.float(), orc.attention(q, k, v, causal=causal), atol=1e-5, rtol=1e-5)
    torch.testing.assert_close(lse.float(), orc.lse(q, k, causal=causal), atol=1e-5, rtol=1e-5)
    visible = nq - max(0, nq - n) if causal else nq  # rows with a visible key
    torch.testing.assert_close(w.sum(-1), torch.full((2, 2), 2.0 * visible, dtype=torch.float64))


def test_attention_weights_closed_forms():
    q, k = torch.zeros(1, 2, 1, 8), torch.randn(1, 1, 5, 8)
    o, lse, w = cor.attention(q, k, k, lens=[4])
    assert w.tolist() == [[[0.5, 0.5, 0.5, 0.5, 0.0]]]
    assert torch.allclose(lse, torch.full((1, 2, 1), math.log(4), dtype=torch.float64))
    assert torch.allclose(o[0, 0, 0], k[0, 0, :4].double().mean(0))


def test_kept():
    s = np.array([5.0, 1.0, 5.0, np.nan, 0.0, 9.0], dtype=np.float32)
    assert cor.kept(s, 6, 6, 0) == [0, 1, 2, 3, 4, 5]
    assert cor.kept(s, 6, 3, 0) == [0, 3, 5]
    assert cor.kept(s, 6, 3, 2) == [3, 4, 5]
    assert cor.kept(s, 5, 3, 1) == [0, 3, 4]
    assert cor.kept(s, 2, 3, 1) == [0, 1]
    assert cor.kept(s, 6, 2, 2) == [4, 5]
    assert cor.kept(np.array([-0.0, 0.0, 0.0], dtype=np.float32), 3, 2, 0) == [0, 1]
