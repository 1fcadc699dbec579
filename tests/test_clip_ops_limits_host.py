"""Sizes past what one launch holds (2^32 - 1 threads) are refused by the
operators around the DiT blocks as unsupported, before any device work."""
from __future__ import annotations

import ctypes

import pytest

from test_clip_ops_host import linear_args, norm_args, sliding


@pytest.mark.parametrize("over", [
    dict(batch=40_000_000, q_len=1, kv_len=1),                       # single tokens
    dict(batch=2, q_len=2**30 // 8, heads=8, kv_heads=1, kv_len=1),  # 16.8 million tiles
])
def test_sliding_attention(hip, over):
    lib = hip.load()
    a = sliding(hip, **over)
    assert lib.sv2_sliding_attention_workspace(ctypes.byref(a)) == hip.SV2_EUNSUPPORTED
    assert lib.sv2_sliding_attention(ctypes.byref(a), None) == hip.SV2_EUNSUPPORTED
    assert b"too many" in lib.sv2_last_error()


@pytest.mark.parametrize("over", [
    dict(images=40_000_000),                                    # held by workgroups
    dict(images=20_000_000, rows=5000, groups=1),     # in runs
])
def test_group_norm(hip, over):
    lib = hip.load()
    assert lib.sv2_group_norm(*norm_args(hip, xi=2**20, yi=2**20, size=1 << 62, **over), None) == hip.SV2_EUNSUPPORTED
    assert b"too many" in lib.sv2_last_error()


@pytest.mark.parametrize("over", [
    dict(rows=2**31 - 1, in_=1, out=1, x_stride=1, w_stride=1, y_stride=1, residual=None),  # tiles of any operands
    dict(rows=1, out=2**31 - 1, in_=8, y_stride=2**31 - 1, residual=None),                  # a stream
    dict(rows=2**31 - 1, out=2**31 - 1, y_stride=2**31, residual=None),                     # tiles of aligned ones
])
def test_linear(hip, over):
    lib = hip.load()
    assert lib.sv2_linear(ctypes.byref(linear_args(hip, **over)), None) == hip.SV2_EUNSUPPORTED
    assert b"too many" in lib.sv2_last_error()
