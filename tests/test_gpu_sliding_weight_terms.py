"""weight_terms = 2 in sv2_sliding_attention's tiles: the error is held to a
bound without the weights' rounding to 16 bits; everything else is as with one
term."""
from __future__ import annotations

import math

import pytest
import torch

import clip_ops_exact as ex
from test_gpu_sliding_attention import TD, check, make, run
from test_gpu_sliding_infinities import plant

pytestmark = pytest.mark.gpu
SHAPES = [
    (60, 60, 4, 4, 128, 60),        # every row sees few keys
    (130, 700, 64, 64, 64, 40),     # two groups of waves, no split
    (200, 3000, 2, 1, 128, 3000),   # splits
    (700, 900, 40, 40, 128, 50),    # one group
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,h,g,d,left", SHAPES)
def test_weights_in_two_terms(hip, device, nq, nk, h, g, d, left, dtype):
    """The bound of the few-row form's test: in place of u sum w|v| for weights
    rounded once, the second term's rounding, u^2 of that."""
    td = TD[dtype]
    q, k, v = make(device, 1, nq, nk, h, g, d, td, seed=nk)
    q = q * 0.25
    scale = d ** -0.5
    want, wl, tol, ltol = ex.sliding_attention(q, k, v, left, 0, 3, scale)
    mass = ex.sliding_attention(q, k, v.abs(), left, 0, 3, scale)[0]
    u = ex.HALF_STEP[td]
    tight = tol - 1.01 * (u - u * u) * mass
    assert (tight > 0).all()
    two, lse = run(hip, q, k, v, left, 0, 3, weight_terms=2)
    ex.close(two, want, tight)
    ex.close(lse, wl, ltol)
    one, lse_one = run(hip, q, k, v, left, 0, 3)
    assert torch.equal(lse, lse_one)
    assert torch.equal(run(hip, q, k, v, left, 0, 3, weight_terms=1)[0], one)
    if left < 100:  # over many keys the roundings average to less than the bound has for the sum
        assert ((one.double() - want).abs() > tight).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,h,g,d,left", SHAPES)
def test_masks_and_values_that_are_not_finite(hip, device, nq, nk, h, g, d, left, dtype):
    q, k, v = make(device, 1, nq, nk, h, g, d, TD[dtype])
    check(hip, q * 8, k * 4, v, left, 0, 3, weight_terms=2)
    plant(v, nk // 2)
    check(hip, q, k, v, nk, 0, 0, weight_terms=2)
    hidden = slice(5, max(5, nk - nq - left))  # between the first tokens and the window
    k[:, hidden] = math.nan
    v[:, hidden] = math.nan
    check(hip, q, k, v, left, 0, 5, weight_terms=2)


def test_few_rows_have_both_anyway(hip, device):
    q, k, v = make(device, 2, 1, 900, 8, 2, 128, torch.bfloat16)
    assert torch.equal(run(hip, q, k, v, 800, 0, 3)[0], run(hip, q, k, v, 800, 0, 3, weight_terms=2)[0])
