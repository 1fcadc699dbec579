"""Float64 definitions of the operators around the DiT blocks (sliding
attention, group norm, linear) and the error bounds their tests use.

u is half a step of the output type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32),
f = 2^-24 one fp32 rounding."""
from __future__ import annotations

import math

import torch

F = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
# |act'| <= 1.13 (gelu; silu 1.1)
SLOPE = 1.13


def rounding(y, dtype):
    return HALF_STEP[dtype] * y.abs() + TINY[dtype]


def visible(nq, nk, left, right, sinks, device):
    p = torch.arange(nk - nq, nk, device=device)[:, None]
    j = torch.arange(nk, device=device)[None]
    return (j <= p + right) & ((j < sinks) | (j >= p - left))


def sliding_attention(q, k, v, left, right, sinks, scale, q_lens=None, kv_lens=None):
    """out, lse, the bound of out's error and of lse's, all float64; rows
    behind a sequence's length are NaN.

    out: rounding of the weights to the inputs' type, u sum w|v|; fp32 sums
    of dim products move a score by at most dim f scale sum|qk| =: s and the
    exponential by 8 f more (the score's two roundings, exp2, the sum), so a
    normalised weight by 2 s + 16 f relative; fp16 weights below 2^-14 of the
    row's largest are off by 2^-25 of it at most; the output's own rounding.
    The sum over n keys adds n f."""
    b, nq_all, h, d = q.shape
    g = h // k.shape[2]
    dtype = q.dtype
    out = torch.full((b, nq_all, h, d), math.nan, dtype=torch.float64, device=q.device)
    lse = torch.full((b, h, nq_all), math.nan, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b):
        nq = nq_all if q_lens is None else int(q_lens[i])
        nk = k.shape[1] if kv_lens is None else int(kv_lens[i])
        if nq == 0:
            continue
        see = visible(nq, nk, left, right, sinks, q.device)
        some = see.any(1) if nk else torch.zeros(nq, dtype=torch.bool, device=q.device)
        for hh in range(h):
            qd = q[i, :nq, hh].double()
            kd, vd = k[i, :nk, hh // g].double(), v[i, :nk, hh // g].double()
            # what no row sees does not count, whatever it holds
            score = torch.where(see, qd @ torch.where(see.any(0)[:, None], kd, 0.0).t() * scale, -math.inf)
            lse_h = torch.logsumexp(score, 1) if nk else torch.full((nq,), -math.inf, device=q.device).double()
            w = torch.where(see, torch.exp(score - lse_h[:, None]), 0.0)
            # values reach the rows that see them only
            fin = torch.where(torch.isfinite(vd), vd, 0.0)
            o = w @ fin
            for value in (math.inf, -math.inf):
                hit = see.double() @ (vd == value).double() > 0
                o = torch.where(hit, o + value, o)
            o = torch.where(see.double() @ torch.isnan(vd).double() > 0, math.nan, o)
            out[i, :nq, hh] = torch.where(some[:, None], o, 0.0)
            lse[i, hh, :nq] = lse_h
            size = qd.abs() @ torch.where(see.any(0)[:, None], kd, 0.0).abs().t() * scale * see
            s = (d * F * size).amax(1) if nk else torch.zeros(nq, device=q.device).double()
            # the fp32 base-2 score and maximum are rounded to 2^-24 of their size
            s = s + (2 * F * (size.amax(1) if nk else 0.0))
            mass = w @ fin.abs()
            small = 2.0 ** -25 * (see.double() @ fin.abs()) * (w.amax(1)[:, None] if nk else 0.0) \
                if dtype == torch.float16 else 0.0
            tol[i, :nq, hh] = (HALF_STEP[dtype] * mass + (2 * s[:, None] + (16 + nk) * F) * mass + small
                               + rounding(o, dtype)) * 1.01
            ltol[i, hh, :nq] = s + (16 + nk) * F + 4 * F * torch.where(some, lse_h, 0.0).abs()
    return out, lse, tol, ltol


def activate(v, act):
    if act == 1:
        return v * torch.sigmoid(v)
    if act == 2:
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    if act == 3:
        return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def act_error(v, act, dtype):
    """Of the activation itself, in fp32: 16 roundings (libm functions, the
    divide); with the 16-bit types exp2 of a rounded exponent, |v| + 4
    roundings of exp(-v) at most (gelu_tanh: of exp(-2u), |2u| <= |v| (1.6 +
    0.08 v^2)), which weighs at most y, or v exp(-|e|) where the exponential
    is small."""
    if act == 0:
        return torch.zeros_like(v)
    e = v.abs() if act != 3 else v.abs() * (1.6 + 0.08 * v * v)
    y = activate(v, act).abs()
    if act == 2 or dtype == torch.float32:
        # the exponent's own rounding enters fp32's tanh form all the same
        return (16 + (2 * e if act == 3 else 0.0)) * F * y + 2.0 ** -126
    return (2 * e + 16) * F * y + 2.0 ** -126


def group_norm(x, groups, gamma, beta, eps, act):
    """y and its bound, float64.  The mean is off by 16 f max|x| at most
    (sums of 8 or 16, then pairwise joins: few roundings each), the variance
    by 64 f of itself and the square of the mean's error, 1 / sqrt by half
    that; the affine step rounds three times."""
    n, rows, c = x.shape
    v = x.double().reshape(n, rows, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = (v - mean).square().mean((1, 3), keepdim=True)
    big = v.abs().amax((1, 3), keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    hat = ((v - mean) * r).reshape(n, rows, c)
    z = hat * g + b
    off = 16 * F * big
    rel = 0.5 * (64 * F * var + off * off) / (var + eps) + 4 * F
    err = ((off * r + rel * ((v - mean) * r).abs()).reshape(n, rows, c) * (g if gamma is None else g.abs())
           + 3 * F * (hat * g).abs() + F * z.abs())
    y = activate(z, act)
    return y, (SLOPE * err + act_error(z, act, x.dtype)) * 1.01 + rounding(y, x.dtype)


def linear(x, w, bias, act, residual):
    """y and its bound, float64.  k products in fp32 sums in any order: k f
    sum|xw|; the bias's and the residual's additions one rounding each."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    err = (x.shape[1] + 1) * F * (xd.abs() @ wd.abs().t())
    if bias is not None:
        z = z + bias.double()
        err = err + F * z.abs()
    y = activate(z, act)
    err = SLOPE * err + act_error(z, act, x.dtype)
    if residual is not None:
        y = y + residual.double()
        err = err + F * y.abs()
    return y, err * 1.01 + rounding(y, x.dtype)


def close(got, want, tol):
    """Equal where not finite, within `tol` elsewhere; NaN in `want` must be
    NaN."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), "infinities in other places"
    d = (got - want).abs()[fine]
    t = tol.expand_as(want)[fine]
    bad = d > t
    if bad.any():
        i = int((d / t).nan_to_num(posinf=0.0).argmax())
        raise AssertionError(f"{int(bad.sum())} of {d.numel()} beyond the bound, worst {float(d[i]):.3e} "
                             f"against {float(t[i]):.3e}")
