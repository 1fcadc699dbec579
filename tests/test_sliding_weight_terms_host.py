"""weight_terms of sv2_sliding_attention: refused outside 0 .. 2; the workspace
does not depend on it."""
from __future__ import annotations

import ctypes

import pytest

from test_clip_ops_host import sliding


@pytest.mark.parametrize("terms", [-1, 3, 100])
def test_refused(hip, terms):
    lib = hip.load()
    a = sliding(hip, weight_terms=terms)
    assert lib.sv2_sliding_attention(ctypes.byref(a), None) == hip.SV2_EINVAL
    assert b"weight_terms" in lib.sv2_last_error()


def test_workspace(hip):
    lib = hip.load()
    sizes = {lib.sv2_sliding_attention_workspace(ctypes.byref(sliding(hip, q_len=200, kv_len=100000, left=99999, weight_terms=t)))
             for t in range(3)}
    assert len(sizes) == 1 and sizes.pop() > 0
