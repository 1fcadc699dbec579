"""Which kernel and tiles sv2_linear takes for the products that the tests of
its forms run: a change of the choice that left a form without a test would
fail here.  Nothing is launched."""
from __future__ import annotations

import ctypes

import pytest

from linear_forms import FEW, TILES, up8
from test_clip_ops_host import P, linear_args


def args(hip, m, k, n, **over):
    a = hip.LinearArgs(m, k, n, hip.F16, 0, P, up8(k), P, up8(k), None, None, 0, P, up8(n))
    for name, v in over.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("size,want", TILES + FEW)
def test_the_tests_reach_the_forms(hip, size, want):
    m, k, n = size
    for dtype in (hip.F16, hip.BF16):
        for act in range(4):
            a = args(hip, m, k, n, dtype=dtype, activation=act)
            assert hip.linear_plan(a, None, None) == want
            a.bias, a.residual, a.residual_stride = P, P, up8(n)
            assert hip.linear_plan(a, None, None) == want


def test_every_form_is_among_them(hip):
    forms = {(w[2] > 0, w[3]) for _, w in TILES}
    assert forms >= {(False, f) for f in hip.TILE_FORMS[:4]} and (True, "128x128") in forms
    assert {w[1] for _, w in FEW} == {16, 64}


def test_layouts_that_leave_the_tiles(hip):
    """An operand out of alignment, or a stride past the 32-bit offsets of a
    tile or of a block of 64 rows."""
    m, k, n = 1217, 1280, 784
    for over in (dict(x=P + 8), dict(w=P + 2), dict(y=P + 8), dict(residual=P + 2, residual_stride=n),
                 dict(x_stride=k + 4), dict(w_stride=k + 1), dict(y_stride=n + 1), dict(x_stride=2**22),
                 dict(w_stride=2**22)):
        kernel, tile, first, form = hip.linear_plan(args(hip, m, k, n, **over), None, None)
        assert (kernel, tile, first, form) == ("any", 64, 0, None), over
    assert hip.linear_plan(args(hip, m, k, n, x_stride=2**22 - 8, w_stride=2**22 - 8), None, None)[0] == "tiles"
    assert hip.linear_plan(args(hip, 64, k, n, x_stride=2**24 - 8, w_stride=2**24 - 8), None, None)[0] == "few"
    assert hip.linear_plan(args(hip, 64, k, n, x_stride=2**24), None, None)[0] == "any"
    assert hip.linear_plan(args(hip, 2100, 133, 2051, x_stride=134), None, None)[:2] == ("any", 128)


def test_plan_argument_checks(hip):
    lib = hip.load()
    plan = (ctypes.c_int * 4)()
    for a in (linear_args(hip, rows=-1), linear_args(hip, x=None), linear_args(hip, rows=0), linear_args(hip, y_stride=1)):
        assert lib.sv2_linear_plan(ctypes.byref(a), plan) == hip.SV2_EINVAL
    assert lib.sv2_linear_plan(ctypes.byref(linear_args(hip)), None) == hip.SV2_EINVAL
    assert lib.sv2_linear_plan(None, plan) == hip.SV2_EINVAL
    assert lib.sv2_linear_plan(ctypes.byref(linear_args(hip, dtype=0)), plan) == hip.SV2_EUNSUPPORTED


def test_plan_of_tensors(hip):
    import torch
    x, w = torch.zeros((40, 64), dtype=torch.float16), torch.zeros((16, 64), dtype=torch.float16)
    y = torch.zeros((40, 16), dtype=torch.float16)
    assert hip.linear_plan(x, w, y) == ("few", 16, 0, None)
    with pytest.raises(ValueError):
        hip.linear_plan(x, w[:, :60], y)
