"""sv2_linear against its definition in float64 with the error bounds of
clip_ops_exact.py: every kernel form, sizes that no tile divides, rows apart
in memory at any alignment, each activation, with and without bias and
residual, values that are not finite beside the operands, graph replays."""
from __future__ import annotations

import math

import pytest
import torch

import clip_ops_exact as ex

pytestmark = pytest.mark.gpu
TD = {"f16": torch.float16, "bf16": torch.bfloat16}


def fenced(shape, pad, shift, gen, dtype, scale=1.0):
    """A [rows, cols] view with `pad` columns behind each row and `shift`
    elements before the first, all of them NaN."""
    rows, cols = shape
    store = torch.full((rows * (cols + pad) + shift + 8,), math.nan, device=gen.device, dtype=dtype)
    view = store[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_(torch.randn(shape, generator=gen, device=gen.device) * scale)
    return store, view


def check(hip, device, m, k, n, dtype, *, act=0, bias=True, residual=True, pad=0, shift=0, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed + m + k + n)
    _, x = fenced((m, k), pad, shift, gen, dtype)
    _, w = fenced((n, k), pad, shift, gen, dtype, 1.0 / math.sqrt(k))
    _, r = fenced((m, n), pad, shift, gen, dtype)
    ys, y = fenced((m, n), pad, shift, gen, dtype)
    y.fill_(math.nan)
    b = torch.randn(n, generator=gen, device=device) if bias else None
    r = r if residual else None
    hip.linear(x, w, y, bias=b, activation=act, residual=r)
    torch.cuda.synchronize()
    want, tol = ex.linear(x, w, b, act, r)
    ex.close(y, want, tol)
    outside = torch.ones_like(ys, dtype=torch.bool)
    outside[shift:shift + m * (n + pad)].view(m, n + pad)[:, :n] = False
    assert torch.isnan(ys[outside]).all(), "something beside y was written"
    return x, w, b, r, y


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [
    (1, 64, 64), (1, 2560, 512), (1, 8, 1), (2, 1, 3), (3, 31, 5), (1, 6912, 257), (7, 1000, 100), (16, 512, 1030),
    (17, 256, 640), (33, 320, 96), (58, 5120, 256), (64, 640, 65), (65, 128, 64), (100, 1001, 77), (129, 72, 130),
    (200, 200, 200), (256, 64, 256), (257, 192, 512), (300, 2560, 384), (513, 100, 700), (1000, 520, 300),
    (2049, 256, 520), (640, 1280, 2560),
])
def test_sizes(hip, device, m, k, n, dtype):
    check(hip, device, m, k, n, TD[dtype], act=1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [
    (1100, 192, 1288), (1500, 264, 776), (3000, 520, 1288), (2600, 1000, 2568), (8200, 64, 264), (4100, 136, 2050),
    (2049, 2560, 640), (1300, 1096, 513),
    (100, 1280, 640), (500, 640, 640), (130, 2560, 2560), (257, 1000, 1024), (65, 640, 10250),
])
@pytest.mark.parametrize("act,residual", [(0, True), (3, False)])
def test_forms_of_many_rows(hip, device, m, k, n, act, residual, dtype):
    """Whole tiles and cut ones of each size, K with and without a rest, and
    rows streamed in blocks of 64."""
    check(hip, device, m, k, n, TD[dtype], act=act, residual=residual)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(2100, 133, 2051), (3000, 70, 3001)])
def test_large_tiles_of_any_alignment(hip, device, m, k, n, dtype):
    check(hip, device, m, k, n, TD[dtype], act=1, pad=1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 320, 192), (40, 320, 192), (600, 320, 256)])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(hip, device, m, k, n, act, bias, residual, dtype):
    check(hip, device, m, k, n, TD[dtype], act=act, bias=bias, residual=residual)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 129, 70), (5, 256, 64), (60, 200, 96), (300, 136, 256), (300, 133, 256)])
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (8, 1), (3, 2), (4, 4), (0, 5)])
def test_strides_and_alignment(hip, device, m, k, n, pad, shift, dtype):
    check(hip, device, m, k, n, TD[dtype], act=3, pad=pad, shift=shift)


@pytest.mark.parametrize("m", [1, 50, 700, 5000])
def test_in_place_residual_and_repeatable(hip, device, m):
    x, w, b, r, y = check(hip, device, m, 512, 250, torch.bfloat16, act=2, pad=6)
    z = r.clone()
    hip.linear(x, w, z, bias=b, activation=2, residual=z)
    torch.cuda.synchronize()
    assert torch.equal(z, y)


@pytest.mark.parametrize("m", [1, 60, 600])
def test_not_finite_stays_in_its_row_and_column(hip, device, m):
    x = torch.randn((m, 192), device=device).to(torch.float16)
    w = (torch.randn((256, 192), device=device) / 14).to(torch.float16)
    w[100, 7] = math.inf
    x[m // 2, 11] = math.nan
    y = torch.empty((m, 256), dtype=torch.float16, device=device)
    hip.linear(x, w, y)
    torch.cuda.synchronize()
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[m // 2] = True
    bad[:, 100] = True
    assert not torch.isfinite(y[bad]).any() and torch.isfinite(y[~bad]).all()


@pytest.mark.parametrize("m,k,n", [(1, 2560, 512), (600, 512, 512)])
def test_streams_and_graph(hip, device, m, k, n):
    x = torch.randn((m, k), device=device).to(torch.float16)
    w = (torch.randn((n, k), device=device) / 50).to(torch.float16)
    y = torch.empty((m, n), dtype=torch.float16, device=device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        hip.linear(x, w, y)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            hip.linear(x, w, y)
    for _ in range(3):
        x.normal_()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = hip.linear(x, w, torch.empty_like(y))
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.parametrize("m", [40, 300])
def test_rows_past_4_gib(hip, device, m):
    step = 2 ** 26
    try:
        store = torch.empty(m * step, dtype=torch.float16, device=device) if m < 100 else \
            torch.empty(m * 2 ** 23, dtype=torch.float16, device=device)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("no room")
    step = store.numel() // m
    x = store.view(m, step)[:, :256]
    x.normal_()
    w = (torch.randn((256, 256), device=device) / 16).to(torch.float16)
    y = store.view(m, step)[:, 4096:4096 + 256]
    hip.linear(x, w, y)
    torch.cuda.synchronize()
    want, tol = ex.linear(x, w, None, 0, None)
    ex.close(y, want, tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("k", [1, 7, 8, 9, 63, 64, 65, 128, 130, 191, 192, 201, 256])
@pytest.mark.parametrize("m,n", [(20, 70), (33, 70), (20, 4100), (130, 70)])
def test_ends_of_k_in_rows_without_alignment(hip, device, m, n, k, dtype):
    """Whole steps, none of them, and every kind of rest."""
    check(hip, device, m, k, n, TD[dtype], act=1, pad=3, shift=1)
