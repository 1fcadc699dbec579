"""Refusals and workspace sizes of the operators around the DiT blocks, on the
host: every bad argument is refused before any device work."""
from __future__ import annotations

import ctypes

import pytest

P = 1 << 20  # a 16-byte aligned address that is never read


def sliding(hip, **over):
    a = hip.SlidingAttnArgs(2, 3, 50, 8, 2, 128, hip.F16, 10, 0, 4, 0.1, P, 3 * 1024, 1024, 128, P, 50 * 256, 256, 128,
                            P, 50 * 256, 256, 128, P, 3 * 1024, 1024, 128)
    a.workspace, a.workspace_bytes = P, 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(batch=-1), -1), (dict(q_len=-1), -1), (dict(kv_len=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1),
    (dict(heads=7), -1), (dict(left=-1), -1), (dict(right=-1), -1), (dict(sinks=-1), -1), (dict(scale=0.0), -1),
    (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(dtype=0), -2),
    (dict(dtype=9), -1), (dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(q_len=2**30, heads=8), -2),
    (dict(kv_len=2**30 + 1), -2), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1),
    (dict(q=P + 8), -1), (dict(k=P + 2), -1), (dict(v=P + 4), -1), (dict(out=P + 8), -1), (dict(lse=P + 2), -1),
    (dict(q_lens=P + 2), -1), (dict(kv_lens=P + 1), -1), (dict(q_token_stride=1025), -1), (dict(k_head_stride=-8), -1),
    (dict(out_batch_stride=4), -1), (dict(k_token_stride=2**24 + 8), -2), (dict(v_token_stride=2**40), -2),
])
def test_sliding_attention_refuses(hip, over, code):
    lib = hip.load()
    a = sliding(hip, **over)
    assert lib.sv2_sliding_attention(ctypes.byref(a), None) == code
    assert b"sv2_sliding_attention" in lib.sv2_last_error()


def test_sliding_attention_nothing_to_do_and_null(hip):
    lib = hip.load()
    assert lib.sv2_sliding_attention(ctypes.byref(sliding(hip, batch=0, q=None)), None) == 0
    assert lib.sv2_sliding_attention(ctypes.byref(sliding(hip, q_len=0, out=None)), None) == 0
    assert lib.sv2_sliding_attention(None, None) == -1
    assert lib.sv2_sliding_attention_workspace(None) == -1
    assert lib.sv2_sliding_attention_workspace(ctypes.byref(sliding(hip, head_dim=80))) == -2


def test_sliding_attention_reads_no_stride_of_one_element(hip):
    """The strides of a batch of one, one token and one head may be anything;
    the refusal below is the workspace's."""
    lib = hip.load()
    a = sliding(hip, batch=1, q_len=1, kv_len=5000, heads=1, kv_heads=1, left=4999, q_batch_stride=1, q_token_stride=3,
                q_head_stride=-1, k_batch_stride=7, k_head_stride=2**60, v_batch_stride=-5, out_head_stride=1,
                workspace=None)
    assert lib.sv2_sliding_attention(ctypes.byref(a), None) == -1
    assert b"workspace" in lib.sv2_last_error()


def test_sliding_attention_workspace(hip):
    lib = hip.load()
    long = sliding(hip, kv_len=100000, left=99999)
    need = lib.sv2_sliding_attention_workspace(ctypes.byref(long))
    assert need > 0
    for over in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=P + 8)):
        a = sliding(hip, kv_len=100000, left=99999, **over)
        assert lib.sv2_sliding_attention(ctypes.byref(a), None) == -1
    # the size depends on the sizes alone
    other = sliding(hip, kv_len=100000, left=99999, q=None, q_token_stride=7)
    assert lib.sv2_sliding_attention_workspace(ctypes.byref(other)) == need


def norm_args(hip, **over):
    a = dict(x=P, xi=640, xr=64, y=P, yi=640, yr=64, dtype=hip.F16, images=2, rows=10, channels=64, groups=8, eps=1e-5,
             gamma=P, beta=P, act=1, ws=P, size=1 << 30)
    a.update(over)
    return [None if v is None else v for v in a.values()]


@pytest.mark.parametrize("over,code", [
    (dict(dtype=7), -1), (dict(images=-1), -1), (dict(rows=-1), -1), (dict(channels=0), -1), (dict(groups=0), -1),
    (dict(groups=7), -1), (dict(channels=16384), -2), (dict(act=4), -1), (dict(act=-1), -1), (dict(eps=-1.0), -1),
    (dict(eps=float("nan")), -1), (dict(x=None), -1), (dict(y=None), -1), (dict(x=P + 1), -1), (dict(y=P + 1), -1),
    (dict(gamma=P + 2), -1), (dict(beta=P + 1), -1), (dict(ws=P + 4), -1), (dict(xr=63), -1), (dict(yr=0), -1),
    (dict(xi=-1), -1), (dict(yi=0), -1), (dict(rows=10**6, ws=None), -1), (dict(rows=10**6, size=100), -1),
    (dict(images=2**31 - 1, groups=64), -2),
])
def test_group_norm_refuses(hip, over, code):
    lib = hip.load()
    assert lib.sv2_group_norm(*norm_args(hip, **over), None) == code
    assert b"sv2_group_norm" in lib.sv2_last_error()


def test_group_norm_nothing_to_do_and_workspace(hip):
    lib = hip.load()
    assert lib.sv2_group_norm(*norm_args(hip, images=0, x=None), None) == 0
    assert lib.sv2_group_norm(*norm_args(hip, rows=0, y=None), None) == 0
    assert lib.sv2_group_norm_workspace(hip.F16, 1, 1 << 20, 64, 8) > 0
    assert lib.sv2_group_norm_workspace(hip.F16, 0, 1 << 20, 64, 8) == 0
    assert lib.sv2_group_norm_workspace(hip.F16, 1, 10, 64, 7) == -1
    assert lib.sv2_group_norm_workspace(hip.F16, 1, 10, 10000, 1) == -2


def linear_args(hip, **over):
    a = hip.LinearArgs(4, 64, 32, hip.BF16, 0, P, 64, P, 64, P, P, 32, P, 32)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(rows=-1), -1), (dict(in_=0), -1), (dict(out=-1), -1), (dict(dtype=0), -2), (dict(dtype=5), -1),
    (dict(activation=4), -1), (dict(activation=-1), -1), (dict(x_stride=63), -1), (dict(w_stride=1), -1),
    (dict(y_stride=31), -1), (dict(residual_stride=31), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1),
    (dict(x=P + 1), -1), (dict(w=P + 1), -1), (dict(y=P + 1), -1), (dict(residual=P + 1), -1), (dict(bias=P + 2), -1),
])
def test_linear_refuses(hip, over, code):
    lib = hip.load()
    assert lib.sv2_linear(ctypes.byref(linear_args(hip, **over)), None) == code
    assert b"sv2_linear" in lib.sv2_last_error()


def test_linear_nothing_to_do_and_null(hip):
    lib = hip.load()
    assert lib.sv2_linear(ctypes.byref(linear_args(hip, rows=0, x=None)), None) == 0
    assert lib.sv2_linear(ctypes.byref(linear_args(hip, out=0, y=None)), None) == 0
    assert lib.sv2_linear(None, None) == -1


@pytest.mark.parametrize("over", [dict(out_token_stride=0), dict(out_head_stride=0), dict(out_batch_stride=0),
                                  dict(scale=3e38)])
def test_sliding_attention_refuses_outputs_that_coincide(hip, over):
    """and a scale that is not finite in base 2."""
    lib = hip.load()
    assert lib.sv2_sliding_attention(ctypes.byref(sliding(hip, **over)), None) == -1
    assert (b"scale" if "scale" in over else b"stride of out") in lib.sv2_last_error()


def test_in_place_with_other_strides_is_refused(hip):
    lib = hip.load()
    for over in (dict(xr=72), dict(yr=72), dict(xi=0)):
        assert lib.sv2_group_norm(*norm_args(hip, **over), None) == -1
        assert b"y is x" in lib.sv2_last_error()
    for over in (dict(y_stride=40), dict(residual_stride=40)):
        assert lib.sv2_linear(ctypes.byref(linear_args(hip, **over)), None) == -1
        assert b"residual is y" in lib.sv2_last_error()


def test_python_functions_refuse_tensors_that_do_not_fit(hip):
    """By type, shape, layout and device, before any call into the library."""
    import torch
    h = torch.float16
    q, k = torch.zeros((1, 2, 4, 64), dtype=h), torch.zeros((1, 9, 2, 64), dtype=h)
    good = dict(q=q, k=k, v=k, out=torch.zeros_like(q), left=3)
    for over in (dict(v=k[:, :8]), dict(k=k.bfloat16()), dict(out=q[:, :1]), dict(q=q.float()),
                 dict(out=q.transpose(-1, -2).contiguous().transpose(-1, -2)),
                 dict(kv_lens=torch.zeros(1, dtype=torch.int64)), dict(q_lens=torch.zeros(2, dtype=torch.int32)),
                 dict(lse=torch.zeros((1, 2, 4))), dict()):  # the last: not on a GPU
        with pytest.raises(ValueError):
            hip.sliding_attention(**{**good, **over})
    x = torch.zeros((2, 5, 8), dtype=h)
    for more in (dict(y=x[:1]), dict(y=x.float()), dict(y=x.clone(), gamma=torch.zeros(8, dtype=h)),
                 dict(y=x.clone(), beta=torch.zeros(7)), dict(y=x.double()), dict(y=x.clone())):
        with pytest.raises(ValueError):
            hip.group_norm(x, groups=2, **more)
    w, y = torch.zeros((6, 8), dtype=h), torch.zeros((5, 6), dtype=h)
    for over in (dict(w=w[:, :7]), dict(y=y[:4]), dict(x=x[0].float()), dict(residual=y[:, :5]), dict(bias=y[0]),
                 dict(w=w.t().contiguous().t()), dict()):
        with pytest.raises(ValueError):
            hip.linear(**{**dict(x=x[0], w=w, y=y), **over})
