"""The few-row form of sv2_sliding_attention multiplies by weights in two 16-bit
terms: its error is held to a bound without the weights' rounding to 16 bits."""
from __future__ import annotations

import pytest
import torch

import clip_ops_exact as ex
from test_gpu_sliding_attention import TD, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,h,g,d", [(1, 60, 16, 16, 128), (1, 60, 40, 20, 64), (4, 500, 8, 1, 128), (2, 3000, 4, 4, 64)])
def test_weights_in_two_terms(hip, device, nq, nk, h, g, d, dtype):
    """clip_ops_exact's bound has u sum w|v| for weights rounded once (u half a
    step of the type).  In two terms the second is the first one's error, at
    most u w, itself rounded: u^2 w, and in fp16 at most 2^-25 of the row's
    largest weight below the normal range, which the bound has already."""
    td = TD[dtype]
    q, k, v = make(device, 1, nq, nk, h, g, d, td, seed=nk)
    q = q * 0.25  # small scores: their own rounding stays below the weights'
    out, _ = run(hip, q, k, v, nk, 0, 0)
    torch.cuda.synchronize()
    scale = d ** -0.5
    want, lse, tol, _ = ex.sliding_attention(q, k, v, nk, 0, 0, scale)
    mass = ex.sliding_attention(q, k, v.abs(), nk, 0, 0, scale)[0]
    u = ex.HALF_STEP[td]
    tight = tol - 1.01 * (u - u * u) * mass
    assert (tight > 0).all()
    ex.close(out, want, tight)
    # weights in one term break it; not over many keys, whose roundings average
    # to less (u / sqrt(keys)) than the bound has for the sum (2^-24 a key)
    if nk > 100:
        return
    see = ex.visible(nq, nk, nk, 0, 0, device)
    once = torch.zeros_like(want)
    for i in range(h):
        score = torch.where(see, q[0, :, i].double() @ k[0, :, i * g // h].double().t() * scale, -torch.inf)
        w = torch.exp(score - score.amax(1, keepdim=True))
        once[0, :, i] = (w.to(td).double() @ v[0, :, i * g // h].double()) / w.sum(1, keepdim=True)
    assert ((once.to(td).double() - want).abs() > tight).any()
