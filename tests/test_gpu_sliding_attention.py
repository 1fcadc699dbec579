"""sv2_sliding_attention against its definition in float64, with the error
bounds of clip_ops_exact.py: lengths around the tiles, windows and first
tokens of every relation to them, shared key heads, both head sizes, strided
layouts, rows that see nothing, values that are not finite where nobody (or
somebody) looks, keys past 4 GiB, split and unsplit forms, graph replays and
other streams."""
from __future__ import annotations

import math

import pytest
import torch

import clip_ops_exact as ex

pytestmark = pytest.mark.gpu
TD = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(device, b, nq, nk, h, g, d, dtype, seed=0, layout="bthd"):
    gen = torch.Generator(device=device).manual_seed(seed)

    def rand(t, heads):
        x = torch.randn((b, t, heads, d), generator=gen, device=device).to(dtype)
        if layout == "bhtd":
            return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        if layout == "padded":
            wide = torch.full((b, t + 1, heads, d + 8), math.nan, device=device).to(dtype)
            wide[:, :t, :, :d] = x
            return wide[:, :t, :, :d]
        return x

    return rand(nq, h), rand(nk, g), rand(nk, g)


def run(hip, q, k, v, left, right, sinks, q_lens=None, kv_lens=None, scale=None, **more):
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), 7.0, device=q.device)
    hip.sliding_attention(q, k, v, out, left=left, right=right, sinks=sinks, q_lens=q_lens, kv_lens=kv_lens, lse=lse,
                          scale=scale, **more)
    return out, lse


def check(hip, q, k, v, left, right, sinks, q_lens=None, kv_lens=None, scale=None, **more):
    out, lse = run(hip, q, k, v, left, right, sinks, q_lens, kv_lens, scale, **more)
    torch.cuda.synchronize()
    s = q.shape[-1] ** -0.5 if scale is None else scale
    want, wl, tol, ltol = ex.sliding_attention(q, k, v, left, right, sinks, s, q_lens, kv_lens)
    for i in range(q.shape[0]):
        n = q.shape[1] if q_lens is None else int(q_lens[i])
        assert (out[i, n:] == 7.0).all() and (lse[i, :, n:] == 7.0).all(), "rows behind the sequence were written"
        ex.close(out[i, :n], want[i, :n], tol[i, :n])
        ex.close(lse[i, :, :n], wl[i, :, :n], ltol[i, :, :n])
    return out, lse


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,nq,nk,h,g,left,right,sinks", [
    (1, 1, 1, 1, 1, 0, 0, 0),
    (1, 1, 700, 4, 4, 300, 0, 5),          # the next token
    (3, 1, 1000, 10, 2, 4000, 0, 0),       # five heads a key head, all of the cache
    (2, 3, 129, 8, 1, 20, 0, 3),
    (1, 63, 63, 2, 1, 10, 0, 0),
    (1, 64, 64, 2, 2, 1000, 0, 64),
    (2, 65, 190, 3, 3, 64, 63, 1),
    (1, 127, 128, 6, 2, 0, 0, 0),          # only itself
    (1, 129, 300, 2, 2, 0, 0, 70),         # itself and the first tokens
    (1, 200, 513, 4, 2, 2**31 - 1, 2**31 - 1, 0),  # everything
    (2, 97, 97, 5, 1, 30, 200, 500),       # more first tokens than tokens
    (1, 300, 1500, 2, 1, 150, 17, 58),
    (1, 40, 25, 2, 2, 100, 0, 4),          # fewer keys than queries: the first see none
    (1, 33, 10, 2, 2, 3, 30, 4),
    (2, 5, 0, 4, 2, 9, 9, 9),              # no keys at all
    (1, 700, 700, 1, 1, 64, 0, 64),
])
def test_lengths_and_windows(hip, device, b, nq, nk, h, g, d, left, right, sinks, dtype):
    q, k, v = make(device, b, nq, nk, h, g, d, TD[dtype], seed=nq + nk)
    check(hip, q, k, v, left, right, sinks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,nq,nk,h,g,left,right,sinks", [
    (3, 1000, 1000, 12, 12, 200, 0, 20),   # more row tiles than CUs
    (2, 700, 900, 40, 10, 300, 50, 3),
    (1, 32, 6000, 2, 2, 6000, 0, 0),       # 32 rows a key head, many splits
    (1, 33, 6000, 2, 2, 6000, 0, 0),       # one more
    (2, 8, 9000, 8, 2, 8000, 7, 100),      # eight tokens of four heads
    (1, 5, 300, 30, 5, 299, 0, 0),         # thirty rows
    (20, 2, 500, 16, 16, 100, 0, 64),      # few splits of many heads
    (1, 129, 40000, 1, 1, 39000, 0, 11),   # two row tiles, many splits
])
def test_forms(hip, device, b, nq, nk, h, g, d, left, right, sinks, dtype):
    q, k, v = make(device, b, nq, nk, h, g, d, TD[dtype], seed=nq)
    check(hip, q, k, v, left, right, sinks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["bhtd", "padded"])
def test_layouts(hip, device, layout, dtype):
    q, k, v = make(device, 2, 50, 140, 4, 2, 128, TD[dtype], layout=layout)
    check(hip, q, k, v, 60, 3, 2)


def test_packed_qkv(hip, device):
    qkv = torch.randn((2, 150, 3, 3, 64), device=device).to(torch.bfloat16)
    check(hip, qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], 40, 0, 9)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,nq,h,g", [(64, 90, 6, 2), (128, 1, 20, 4), (128, 70, 2, 2), (128, 2, 4, 4)])
def test_ragged(hip, device, d, nq, h, g, dtype):
    q, k, v = make(device, 6, nq, 400, h, g, d, TD[dtype])
    q_lens = torch.tensor([nq, 0, 1, nq // 2, nq, nq], dtype=torch.int32, device=device)
    kv_lens = torch.tensor([400, 10, 399, 0, 1, 65], dtype=torch.int32, device=device)
    for i, n in enumerate(kv_lens.tolist()):
        k[i, n:] = math.nan
        v[i, n:] = math.inf
    check(hip, q, k, v, 100, 5, 7, q_lens, kv_lens)
    # lengths beyond the tensors count as theirs
    out, lse = run(hip, q, k[:, :65], v[:, :65], 100, 5, 7,
                   torch.full_like(q_lens, 10**6), torch.full_like(kv_lens, -5))
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,h,g,d", [(1, 4, 2, 128), (4, 8, 1, 64), (150, 2, 1, 128), (150, 2, 2, 64)])
def test_values_that_are_not_finite(hip, device, nq, h, g, d, dtype):
    """Keys and values between the first tokens and the window hold anything;
    a value that some rows see reaches those rows only."""
    q, k, v = make(device, 1, nq, 500, h, g, d, TD[dtype])
    left, sinks = 90, 10
    lo = 500 - nq - left
    k[:, sinks:lo] = math.nan
    v[:, sinks:lo:2] = math.nan
    v[:, sinks + 1:lo:2] = -math.inf
    check(hip, q, k, v, left, 0, sinks)
    # seen by the later rows: the last keys
    v[0, 499, 0, 3] = math.inf
    v[0, 498, 0, 3] = -math.inf
    v[0, 498, 0, 5] = math.nan
    v[0, 497, 0, 40] = -math.inf
    v[0, 2, 0, 7] = math.inf  # a first token: seen by all
    check(hip, q, k, v, left, 0, sinks)


@pytest.mark.parametrize("nq,h", [(40, 2), (700, 40)])
def test_values_that_are_not_finite_in_every_tile(hip, device, nq, h):
    """Windows so narrow that every tile is masked, with a value of each kind
    every few keys."""
    q, k, v = make(device, 1, nq, nq + 300, h, h, 128, torch.bfloat16)
    v[:, 5::67, :, 3] = math.inf
    v[:, 9::71, :, 3] = -math.inf
    v[:, 40::97, :, 60] = math.nan
    v[:, 50::61] = math.inf
    check(hip, q, k, v, 20, 0, 2)


@pytest.mark.parametrize("nq", [1, 40])
def test_scores_that_are_not_finite(hip, device, nq):
    """A row whose only visible scores are -Inf counts as empty; +Inf and NaN
    scores give NaN, as the softmax does."""
    q = torch.ones((1, nq, 2, 64), dtype=torch.float16, device=device)
    k = torch.full((1, 100, 2, 64), -math.inf, dtype=torch.float16, device=device)
    v = torch.ones_like(k)
    out, lse = run(hip, q, k, v, 1000, 0, 0)
    assert (out == 0).all() and (lse == -math.inf).all()
    v[0, 3] = math.inf
    assert (run(hip, q, k, v, 1000, 0, 0)[0] == 0).all()
    v[0, 3] = 1.0
    k[0, 3] = math.inf
    out, lse = run(hip, q, k, v, 1000, 0, 0)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    k[0, 3] = math.nan
    out, _ = run(hip, q, k, v, 1000, 0, 0)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_large_and_equal_scores(hip, device, dtype):
    q, k, v = make(device, 1, 100, 700, 2, 2, 128, TD[dtype])
    check(hip, q * 8, k * 4, v, 500, 0, 3)  # a row attends to few keys
    check(hip, q * 0, k, v, 500, 0, 3)      # to all of them alike
    check(hip, q, k, v, 500, 0, 3, scale=1e-3)
    # rising scores: the running maximum moves with every tile
    k2 = k * torch.linspace(0, 6, 700, device=device).to(k.dtype)[None, :, None, None]
    check(hip, q.abs(), k2.abs(), v, 700, 0, 0)


@pytest.mark.parametrize("nq", [1, 60])
def test_keys_past_4_gib(hip, device, nq):
    step = 2 ** 23
    rows = 300
    try:
        store = torch.empty(rows * step, dtype=torch.float16, device=device)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("no room for a 5 GB cache")
    cache = store.view(1, rows, step)
    q, k, v = make(device, 1, nq, rows, 2, 1, 128, torch.float16)
    cache[:, :, :128] = k[:, :, 0]
    cache[:, :, 1024:1152] = v[:, :, 0]
    ks, vs = cache[:, :, None, :128], cache[:, :, None, 1024:1152]
    check(hip, q, ks, vs, 100, 0, 10)


def test_repeatable_and_workspace(hip, device):
    q, k, v = make(device, 2, 9, 3000, 4, 2, 128, torch.bfloat16)
    a = run(hip, q, k, v, 2500, 0, 4)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device=device)  # NaN patterns
    b = run(hip, q, k, v, 2500, 0, 4, workspace=ws)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(hip.Sv2Error):
        run(hip, q, k, v, 2500, 0, 4, workspace=ws[:16])


def test_streams_and_graph(hip, device):
    """Two calls on two streams with workspaces of their own; a captured call
    follows the lengths and inputs written before each replay."""
    q, k, v = make(device, 2, 1, 2000, 8, 2, 128, torch.float16)
    kv = torch.tensor([2000, 1500], dtype=torch.int32, device=device)
    want = run(hip, q, k, v, 1900, 0, 8, kv_lens=kv)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2):
        with torch.cuda.stream(s):
            got.append(run(hip, q, k, v, 1900, 0, 8, kv_lens=kv))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    out = torch.zeros_like(q)
    ws = torch.empty(16 << 20, dtype=torch.uint8, device=device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s1):
        hip.sliding_attention(q, k, v, out, left=1900, sinks=8, kv_lens=kv, workspace=ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s1):
            hip.sliding_attention(q, k, v, out, left=1900, sinks=8, kv_lens=kv, workspace=ws)
    for n in (2000, 1, 0, 777):
        kv.fill_(n)
        q.normal_()
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager, _ = run(hip, q, k, v, 1900, 0, 8, kv_lens=kv)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,h,d", [(1, 500, 4, 128), (1, 9000, 2, 64), (200, 700, 2, 128), (300, 300, 300, 64)])
def test_scores_of_any_size(hip, device, nq, nk, h, d, dtype):
    """Scores in the thousands and up to 2^40, products of powers of two and
    small integers that fp32 holds: one key of each row carries all the weight,
    or two equal ones share it, so out is their values (half the sum, rounded)
    and lse the score."""
    gen = torch.Generator(device=device).manual_seed(nk)
    td = TD[dtype]
    for power in (2.0 ** 12, 2.0 ** 20, 2.0 ** 32):
        a = torch.randint(-120, 121, (nk,), generator=gen, device=device).float()
        a[torch.randint(0, nk, (1,), generator=gen, device=device)] = 125.0
        q = torch.zeros((1, nq, h, d), device=device)
        k = torch.zeros((1, nk, h, d), device=device)
        q[..., 0] = power ** 0.5
        k[0, :, :, 0] = a[:, None] * power ** 0.5
        v = torch.randn((1, nk, h, d), generator=gen, device=device).to(td)
        q, k = q.to(td), k.to(td)
        if not torch.isfinite(k).all():
            assert td is torch.float16
            k[0, :, :, 0] = a[:, None].to(td)
            q[..., 0] = 2.0 ** 15
        score = q[0, 0, 0, 0].double() * k[0, :, 0, 0].double()
        out, lse = run(hip, q, k, v, nk, 0, 0, scale=4.0)
        for i in range(nq):
            seen = score[:nk - nq + i + 1]
            top = torch.nonzero(seen == seen.max())[:, 0]
            if len(top) > 2:
                continue
            # the mean of one or two values: exact in float64 and, but for the
            # output's rounding, in fp32
            want = v[0, top].double().mean(0).to(td)
            assert torch.equal(out[0, i], want), (power, i)
            far = 4.0 * float(seen.max()) + math.log(len(top))
            assert (lse[0, :, i].double() - far).abs().max() <= abs(far) * 2.0 ** -22
