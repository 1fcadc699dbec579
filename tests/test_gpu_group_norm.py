"""sv2_group_norm against its definition in float64 with the error bounds of
clip_ops_exact.py: both forms (rows held by a workgroup, rows in runs), odd
widths and alignments, means far from zero, constant groups, values that are
not finite, strides past 4 GiB, in place, graph replays."""
from __future__ import annotations

import math

import pytest
import torch

import clip_ops_exact as ex

pytestmark = pytest.mark.gpu
TD = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def affine(c, device, seed=1):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (1 + 0.3 * torch.randn(c, generator=gen, device=device), 0.3 * torch.randn(c, generator=gen, device=device))


def check(hip, x, groups, gamma, beta, eps=1e-5, act=0, y=None):
    want, tol = ex.group_norm(x, groups, gamma, beta, eps, act)
    y = torch.full(x.shape, math.nan, dtype=x.dtype, device=x.device) if y is None else y
    hip.group_norm(x, y, groups, gamma=gamma, beta=beta, eps=eps, activation=act)
    torch.cuda.synchronize()
    ex.close(y, want, tol)
    return y


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,rows,groups,width", [
    (1, 1, 1, 1), (2, 1, 4, 1), (1, 2, 1, 8), (3, 5, 32, 16), (2, 480, 32, 16), (1, 257, 8, 3), (2, 1000, 32, 10),
    (1, 7, 1, 513), (1, 4096, 32, 4), (2, 5000, 16, 8), (1, 3001, 1, 64), (1, 9001, 7, 5), (1, 64, 2, 4096),
    (1, 700, 8, 1000), (4, 1100, 1, 1), (1, 100000, 1, 8), (1, 2500, 4, 96),
])
def test_sizes(hip, device, n, rows, groups, width, dtype):
    gen = torch.Generator(device=device).manual_seed(rows)
    c = groups * width
    x = torch.randn((n, rows, c), generator=gen, device=device) + torch.randn(c, generator=gen, device=device)
    g, b = affine(c, device)
    check(hip, x.to(TD[dtype]), groups, g, b, act=1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("rows", [100, 6000])
def test_activations(hip, device, act, rows, dtype):
    x = torch.randn((2, rows, 64), device=device).to(TD[dtype])
    g, b = affine(64, device)
    check(hip, x, 8, g * 6, b, act=act)
    check(hip, x, 8, None, b, act=act)
    check(hip, x, 8, g, None, act=act)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [60, 9000])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (1, 0), (8, 1), (8, 3)])
def test_strides_and_alignment(hip, device, rows, pad, shift, dtype):
    """Rows apart in memory; `shift`: the first element away from a 16-byte
    boundary.  What lies between the rows stays."""
    c, n = 48, 2
    gen = torch.Generator(device=device).manual_seed(5)
    xs = torch.randn(n * rows * (c + pad) + 8, generator=gen, device=device).to(TD[dtype])
    ys = torch.full_like(xs, 5.0)
    x, y = (t[shift:shift + n * rows * (c + pad)].view(n, rows, c + pad)[:, :, :c] for t in (xs, ys))
    g, b = affine(c, device)
    check(hip, x, 6, g, b, act=1, y=y)
    if pad:
        assert (ys[shift:shift + n * rows * (c + pad)].view(n, rows, c + pad)[:, :, c:] == 5.0).all()
    assert (ys[:shift] == 5.0).all() and (ys[shift + n * rows * (c + pad):] == 5.0).all()


@pytest.mark.parametrize("rows", [50, 20000])
def test_images_interleaved(hip, device, rows):
    """[rows, images, channels] seen as [images, rows, channels]."""
    x = torch.randn((rows, 3, 32), device=device).permute(1, 0, 2)
    y = torch.empty((rows, 3, 32), device=device).permute(1, 0, 2)
    check(hip, x, 4, None, None, y=y)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [300, 30000])
def test_means_far_from_zero(hip, device, rows, dtype):
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.randn((2, rows, 32), generator=gen, device=device)
    check(hip, (x + 1000.0).to(TD[dtype]), 4, None, None)
    # a border of zeros, then values around 500
    x = x + 500.0
    x[:, :40] = 0.0
    check(hip, x.to(TD[dtype]), 4, None, None, act=1)
    # one group of constants
    x[:, :, :8] = 3.25
    check(hip, x.to(TD[dtype]), 4, None, None)


@pytest.mark.parametrize("rows", [100, 30000])
def test_not_finite_stays_in_its_group(hip, device, rows):
    x = torch.randn((2, rows, 32), device=device)
    x[0, 17, 9] = math.nan
    x[1, 3, 31] = math.inf
    y = torch.empty_like(x)
    hip.group_norm(x, y, 4)
    want, tol = ex.group_norm(x, 4, None, None, 1e-5, 0)
    bad = torch.zeros((2, 1, 4), dtype=torch.bool, device=device)
    bad[0, 0, 1] = bad[1, 0, 3] = True
    bad = bad.repeat_interleave(8, 2).expand_as(x)
    assert torch.isnan(y[bad]).all()
    ex.close(y[~bad], want[~bad], tol[~bad])


@pytest.mark.parametrize("rows", [100, 30000])
def test_in_place_repeatable_and_graph(hip, device, rows):
    x = torch.randn((2, rows, 96), device=device).to(torch.bfloat16)
    g, b = affine(96, device)
    y = check(hip, x, 8, g, b, act=1)
    ws = torch.full((8 << 20,), 0xFF, dtype=torch.uint8, device=device)
    z = x.clone()
    hip.group_norm(z, z, 8, gamma=g, beta=b, activation=1, workspace=ws)
    assert torch.equal(y, z)
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        hip.group_norm(x, out, 8, gamma=g, beta=b, activation=1, workspace=ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            hip.group_norm(x, out, 8, gamma=g, beta=b, activation=1, workspace=ws)
    for _ in range(3):
        x.normal_()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = hip.group_norm(x, torch.empty_like(x), 8, gamma=g, beta=b, activation=1)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("rows", [64, 5000])
def test_images_past_4_gib(hip, device, rows):
    step = 2 ** 31 + 2 ** 20
    try:
        store = torch.empty(step + rows * 64, dtype=torch.float16, device=device)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("no room")
    x = torch.as_strided(store, (2, rows, 64), (step, 64, 1))
    x.normal_()
    y = torch.empty((2, rows, 64), dtype=torch.float16, device=device)
    check(hip, x, 8, None, None, y=y)
    src = x.contiguous()
    z = torch.as_strided(store, (2, rows, 64), (step, 64, 1))
    hip.group_norm(src, z, 8)
    assert torch.equal(z, y)


def test_workspace_refused(hip, device):
    x = torch.randn((1, 40000, 64), device=device)
    with pytest.raises(hip.Sv2Error):
        hip.group_norm(x, torch.empty_like(x), 8, workspace=torch.empty(16, dtype=torch.uint8, device=device))
