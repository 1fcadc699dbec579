"""sv2_sliding_attention where values that are not finite are seen by every
row of a tile: an infinity or NaN reaches the rows that see it, whatever its
weight and wherever its key stands, in the few-row form, the tiles, the
splits and their joins."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sliding_attention import TD, check, make, run

pytestmark = pytest.mark.gpu


def plant(v, at):
    """Values of each kind in dims of their own from key `at` on."""
    v[:, at, :, 3] = math.inf
    v[:, at + 1, :, 9] = -math.inf
    v[:, at + 2, :, 17] = math.nan
    v[:, at + 3, :, 40] = math.inf
    v[:, at + 5, :, 40] = -math.inf
    v[:, at + 6, 0, 41] = math.inf


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,nk,h,g,at", [
    (1, 512, 1, 1, 200),     # one split a tile
    (1, 700, 4, 2, 40),
    (1, 9000, 2, 2, 4000),   # many splits
    (4, 600, 8, 1, 300),     # all 32 rows
    (1, 64, 300, 300, 10),   # no split: the waves' join writes out
])
def test_few_rows_see_all(hip, device, nq, nk, h, g, at, d, dtype):
    """Every key but the last few is seen by every row: tiles without a mask."""
    q, k, v = make(device, 1, nq, nk, h, g, d, TD[dtype], seed=nk)
    plant(v, at)
    out, _ = check(hip, q, k, v, nk, 0, 0)
    assert (out[..., 3] == math.inf).all() and (out[..., 9] == -math.inf).all() and torch.isnan(out[..., 17]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk", [(1, 512), (2, 9000)])
def test_few_rows_whose_weight_is_lost(hip, device, nq, nk, dtype):
    """Scores that rise until a weight of the first keys is 0 in fp32, in one
    stream and across splits: the sums so far are scaled by 0, the infinities
    among them stay."""
    q, k, v = make(device, 1, nq, nk, 2, 2, 128, TD[dtype], seed=1)
    q, k = q.abs() + 0.5, (k.abs() + 0.5) * torch.linspace(0, 4, nk, device=device).to(k.dtype)[None, :, None, None]
    plant(v, 20)
    plant(v, nk // 2)
    check(hip, q, k, v, nk, 0, 0)
    # and fall again
    check(hip, q, k.flip(1), v, nk, 0, 0)
    # seen, but of no score at all in the first half
    q[..., 0] = 1.0
    k[:, :nk // 2, :, 0] = -math.inf
    out, _ = run(hip, q, k, v, nk, 0, 0)
    assert (out[..., 3] == math.inf).all() and (out[..., 9] == -math.inf).all() and torch.isfinite(out[..., 20:39]).all()


def lost(device, nq, nk, h, g, d, dtype):
    """Scores so far apart that most weights are 0 in 16 bits, many in fp32:
    small ones, a few large keys, and rising ones."""
    q, k, v = make(device, 1, nq, nk, h, g, d, TD[dtype], seed=nk)
    q, k = q.abs() + 0.5, k.abs() + 0.5
    for far in (2.0, 8.0):
        rise = torch.linspace(0, far, nk, device=device).to(k.dtype)[None, :, None, None]
        yield q, k * rise, v.clone()
        yield q, k * rise.flip(1), v.clone()
    k = k * 0.125
    k[:, 5::101] *= 16.0
    yield q, k, v


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,h,g,d", [
    (200, 1000, 2, 2, 128),   # two groups of waves, splits
    (60, 6000, 2, 1, 64),     # many splits
    (130, 700, 64, 64, 64),   # two groups, no split
    (700, 900, 40, 40, 128),  # one group
])
def test_tiles_see_all(hip, device, nq, nk, h, g, d, dtype):
    """Values of each kind at keys that every row sees, with weights that
    matter and weights that are lost."""
    at = (nk - nq) // 2
    q, k, v = make(device, 1, nq, nk, h, g, d, TD[dtype])
    plant(v, at)
    out, _ = check(hip, q, k, v, nk, 0, 0)
    assert (out[..., 3] == math.inf).all() and torch.isnan(out[..., 17]).all()
    for q, k, v in lost(device, nq, nk, h, g, d, dtype):
        plant(v, at)
        plant(v, 8)
        out, _ = check(hip, q, k, v, nk, 0, 0)
        assert (out[..., 3] == math.inf).all() and (out[..., 9] == -math.inf).all() and torch.isnan(out[..., 17]).all()
        # and where some rows see them only
        plant(v, nk - nq + 20)
        check(hip, q, k, v, nq // 2 + 100, 0, 12)


@pytest.mark.parametrize("nq,h", [(150, 2), (700, 40)])
def test_rows_that_are_not_finite_stay_alone(hip, device, nq, h):
    """A row of NaN beside infinite values: its outputs are NaN, the others'
    as they were."""
    q, k, v = make(device, 1, nq, nq + 200, h, h, 64, torch.float16)
    plain, _ = run(hip, q, k, v, 4000, 0, 0)
    q2 = q.clone()
    q2[0, 77, 1] = math.nan
    out, _ = run(hip, q2, k, v, 4000, 0, 0)
    assert torch.isnan(out[0, 77, 1]).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, 77, 1] = False
    assert torch.equal(out[keep], plain[keep])
    plant(v, 100)
    out, _ = run(hip, q2, k, v, 4000, 0, 0)
    assert torch.isnan(out[0, 77, 1]).all()
    want, _ = check(hip, q, k, v, 4000, 0, 0)
    assert torch.equal(out[keep].view(torch.int16), want[keep].view(torch.int16))
