"""sv2_linear's forms for operands in aligned pieces -- every tile form of the
persistent kernel, its two-launch plan, and the stream in blocks of 64 rows --
against the float64 definition and the error bounds of clip_ops_exact.py.
linear_forms.py lists the sizes, and test_linear_forms_host.py holds each to
the form it is meant for.  Row strides are rounded up to multiples of 8
elements, with NaN behind the rows: k and n are cut inside a piece of 16 bytes."""
from __future__ import annotations

import math

import pytest
import torch

import clip_ops_exact as ex
from linear_forms import FEW, TILES, sizes, up8

pytestmark = pytest.mark.gpu
TD = {"f16": torch.float16, "bf16": torch.bfloat16}
# (activation, bias, residual): each activation with and without either
EPILOGUES = [(0, False, False), (0, True, True), (1, True, False), (1, False, True), (2, False, True), (2, True, False),
             (3, True, True), (3, False, False)]
ONE_OF_EACH = [TILES[1][0], TILES[3][0], TILES[5][0], TILES[7][0], TILES[9][0], FEW[2][0], FEW[3][0], FEW[5][0]]


def fenced(rows, cols, stride, dtype, device, fill=math.nan):
    """(storage, view [rows, cols]) with `stride` elements from row to row and
    8 more behind the last, all `fill`."""
    store = torch.full((rows * stride + 8,), fill, device=device, dtype=dtype)
    return store, store[:rows * stride].view(rows, stride)[:, :cols]


def operands(device, m, k, n, dtype, bias=True, residual=True, pad=0, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed + m + k + n)

    def rand(rows, cols, scale=1.0):
        view = fenced(rows, cols, up8(cols) + pad, dtype, device)[1]
        view.copy_(torch.randn((rows, cols), generator=gen, device=device) * scale)
        return view

    x, w, r = rand(m, k), rand(n, k, 1.0 / math.sqrt(k)), rand(m, n)
    return x, w, torch.randn(n, generator=gen, device=device) if bias else None, r if residual else None


def check(hip, device, size, dtype, act, bias, residual, pad=0):
    m, k, n = size
    x, w, b, r = operands(device, m, k, n, dtype, bias, residual, pad)
    ys, y = fenced(m, n, up8(n) + pad, dtype, device)
    assert hip.linear_plan(x, w, y, bias=b, residual=r) == dict(TILES + FEW)[size]
    hip.linear(x, w, y, bias=b, activation=act, residual=r)
    torch.cuda.synchronize()
    ex.close(y, *ex.linear(x, w, b, act, r))
    y.fill_(math.nan)
    assert torch.isnan(ys).all(), "something beside y was written"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act,bias,residual", EPILOGUES)
@pytest.mark.parametrize("size", sizes(TILES), ids=lambda s: "x".join(map(str, s)))
def test_tiles(hip, device, size, act, bias, residual, dtype):
    check(hip, device, size, TD[dtype], act, bias, residual)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act,bias,residual", EPILOGUES)
@pytest.mark.parametrize("size", sizes(FEW), ids=lambda s: "x".join(map(str, s)))
def test_stream(hip, device, size, act, bias, residual, dtype):
    check(hip, device, size, TD[dtype], act, bias, residual)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", sizes(TILES + FEW), ids=lambda s: "x".join(map(str, s)))
def test_rows_apart(hip, device, size, dtype):
    check(hip, device, size, TD[dtype], 3, True, True, pad=24)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m", [20, 60, 300, 1400, 6000])
@pytest.mark.parametrize("n", [513, 1283, 2050])
@pytest.mark.parametrize("k", [1, 9, 65, 70, 129, 133, 1001])
def test_cut_rows(hip, device, m, k, n, residual, dtype):
    """k and n inside a piece, whatever form takes them."""
    x, w, b, r = operands(device, m, k, n, TD[dtype], True, residual)
    ys, y = fenced(m, n, up8(n), TD[dtype], device)
    assert hip.linear_plan(x, w, y, bias=b, residual=r)[0] != "any" or k < 64
    hip.linear(x, w, y, bias=b, activation=1, residual=r)
    torch.cuda.synchronize()
    ex.close(y, *ex.linear(x, w, b, 1, r))
    y.fill_(math.nan)
    assert torch.isnan(ys).all(), "something beside y was written"


@pytest.mark.parametrize("size", ONE_OF_EACH, ids=lambda s: "x".join(map(str, s)))
def test_in_place_residual(hip, device, size):
    m, k, n = size
    x, w, b, r = operands(device, m, k, n, torch.bfloat16)
    y = fenced(m, n, up8(n), torch.bfloat16, device)[1]
    hip.linear(x, w, y, bias=b, activation=1, residual=r)
    store, z = fenced(m, n, up8(n), torch.bfloat16, device)
    for _ in range(3):
        z.copy_(r)
        hip.linear(x, w, z, bias=b, activation=1, residual=z)
        torch.cuda.synchronize()
        assert torch.equal(z, y)
    z.fill_(math.nan)
    assert torch.isnan(store).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", ONE_OF_EACH, ids=lambda s: "x".join(map(str, s)))
def test_not_finite_stays_in_its_row_and_column(hip, device, size, dtype):
    """A NaN and an infinity in the last piece of a row of x and of w, and in
    the residual; the neighbours are those of finite operands."""
    m, k, n = size
    x, w, b, r = operands(device, m, k, n, TD[dtype])
    plain, y = (fenced(m, n, up8(n), TD[dtype], device)[1] for _ in range(2))
    hip.linear(x, w, plain, bias=b, residual=r)
    x[m // 2, k - 1] = math.nan
    w[n - 2, k - 2] = math.inf
    w[n // 3, 1] = -math.inf
    r[0, n // 2] = math.nan
    hip.linear(x, w, y, bias=b, residual=r)
    torch.cuda.synchronize()
    bad = torch.zeros((m, n), dtype=torch.bool, device=device)
    bad[m // 2] = True
    bad[:, n - 2] = True
    bad[:, n // 3] = True
    bad[0, n // 2] = True
    assert not torch.isfinite(y[bad]).any()
    assert torch.equal(y[~bad], plain[~bad]) and torch.isfinite(plain).all()


@pytest.mark.parametrize("size", ONE_OF_EACH, ids=lambda s: "x".join(map(str, s)))
def test_captured(hip, device, size):
    m, k, n = size
    x, w, b, r = operands(device, m, k, n, torch.float16)
    y = fenced(m, n, up8(n), torch.float16, device)[1]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        hip.linear(x, w, y, bias=b, activation=3, residual=r)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            hip.linear(x, w, y, bias=b, activation=3, residual=r)
    for _ in range(3):
        x.normal_()
        r.normal_()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = hip.linear(x, w, fenced(m, n, up8(n), torch.float16, device)[1], bias=b, activation=3, residual=r)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.parametrize("far", ["x", "w"])
@pytest.mark.parametrize("size,stride", [
    ((64, 200, 60), 2**24 - 8), ((17, 333, 64), 2**24 - 8),       # a stream: rows of a block within 2 GiB
    ((640, 1280, 2560), 2**22 - 8), ((2600, 1000, 2568), 2**22 - 8), ((1352, 200, 1480), 2**22 - 8),  # tiles
], ids=str)
def test_rows_far_apart(hip, device, size, stride, far):
    """Row strides just under what the kernels' 32-bit offsets hold."""
    m, k, n = size
    x, w, b, r = operands(device, m, k, n, torch.bfloat16)
    rows = m if far == "x" else n
    try:
        store = torch.empty((rows - 1) * stride + up8(k), dtype=torch.bfloat16, device=device)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("no room")
    wide = torch.as_strided(store, (rows, k), (stride, 1))
    wide.copy_(x if far == "x" else w)
    y, z = (fenced(m, n, up8(n), torch.bfloat16, device)[1] for _ in range(2))
    hip.linear(x, w, y, bias=b, residual=r)
    fx, fw = (wide, w) if far == "x" else (x, wide)
    assert hip.linear_plan(fx, fw, z, bias=b, residual=r) == hip.linear_plan(x, w, y, bias=b, residual=r)
    hip.linear(fx, fw, z, bias=b, residual=r)
    torch.cuda.synchronize()
    ex.close(z, *ex.linear(x, w, b, 0, r))
    assert torch.equal(z, y)
