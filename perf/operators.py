"""Operators around the DiT blocks, in their plain form and as the library has them.

Three operators that a clip of many frames needs beside the windowed
attention: the attention of a chunk of tokens over a cache with a sliding
window and first tokens that stay visible, the per-frame group normalisation
with its activation of a channels-last video, and the matrix product with its
bias, activation and residual.  Sizes are the library's own where it has them
(20 heads of 128, hidden size 2560, MLP 6912, 58 text tokens of 5120 channels,
token grids 2x16x30 and 6x45x80), else generic.

  own                 False: the plain forms; True: the library's kernels
  listed()            the named cases
  draw(rng)           one more case from the same ranges
  prepare(case, seed) inputs and weights on the GPU
  run(state)          one pass through an operator
  work(case)          the bytes and operations the pass cannot do without
  exact(case, seed)   the same outputs in float64
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


# ---------------------------------------------------------------- the cases


def _attention(batch, q, kv, heads, kv_heads, dim, left, right, sinks, dtype, **more):
    """`q` rows and `kv` cache rows of sequence 0; each later sequence has
    `q_step` and `kv_step` fewer.  `cap`: rows of the cache.  `packed`: q, k
    and v are slices of one [rows, 3, heads, dim] tensor."""
    case = dict(op="attention", batch=batch, q=q, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, left=left,
                right=right, sinks=sinks, dtype=dtype, cap=kv, q_step=0, kv_step=0, lse=False, packed=False)
    case.update(more)
    return case


def _norm(frames, rows, groups, width, dtype, **more):
    """`frames` of `rows` pixels of groups * width channels; `pad`: unused
    channels behind each pixel's."""
    case = dict(op="norm", frames=frames, rows=rows, groups=groups, width=width, dtype=dtype, act="silu", affine=True,
                pad=0)
    case.update(more)
    return case


def _linear(rows, k, n, dtype, **more):
    """y [rows, n] of x [rows, k]; `pad`: unused columns behind each row of x,
    the residual and y."""
    case = dict(op="linear", rows=rows, k=k, n=n, dtype=dtype, act="none", bias=True, residual=False, pad=0)
    case.update(more)
    return case


def listed():
    return [
        # the next token of one sequence: latency, one long cache
        _attention(1, 1, 4058, 20, 20, 128, 1919, 0, 58, "f16", cap=4224, name="attn_token_f16"),
        # the next token of sixteen sequences of unlike lengths that share
        # key heads: reads the window of every cache
        _attention(16, 1, 16000, 20, 4, 128, 8191, 0, 64, "bf16", cap=16384, kv_step=901, name="attn_tokens_bf16"),
        # a new frame of a 480x256 clip (480 tokens, which see each other)
        # over the text tokens and the last four frames
        _attention(1, 480, 4378, 20, 20, 128, 1920, 479, 58, "f16", cap=4858, name="attn_frame_f16"),
        # three chunks of unlike lengths, narrow heads, the log-sums wanted
        _attention(3, 777, 5003, 12, 3, 64, 1000, 100, 4, "f16", cap=5120, q_step=201, kv_step=1333, lse=True,
                   name="attn_ragged_f16"),
        # a whole prompt: 58 text tokens and 8192 more from one packed qkv
        _attention(1, 8250, 8250, 20, 20, 128, 2047, 0, 58, "bf16", packed=True, name="attn_prompt_bf16"),
        # one small frame: launch-bound
        _norm(1, 480, 32, 16, "f16", name="norm_frame_f16"),
        # three frames of 45x80 in fp32, ten channels a group, no activation
        _norm(3, 3600, 32, 10, "f32", act="none", name="norm_odd_f32"),
        # three frames of 360x640 with 256 channels: memory-bound
        _norm(3, 230400, 32, 8, "bf16", name="norm_clip_bf16"),
        # one row through the time MLP's last product
        _linear(1, 2560, 15360, "f16", act="silu", name="linear_token_f16"),
        # the text projection: 58 rows of 5120 channels
        _linear(58, 5120, 2560, "bf16", name="linear_text_bf16"),
        # sizes that no tile divides, rows apart in memory
        _linear(1999, 1001, 777, "f16", act="gelu", residual=True, pad=7, name="linear_odd_f16"),
        # the tokens of a 720p clip through an MLP's first product
        _linear(21658, 2560, 6912, "bf16", act="gelu_tanh", name="linear_clip_bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attention", "norm", "linear"))
    if op == "attention":
        while True:
            dim = rng.choice((64, 128))
            kv_heads = rng.choice((1, 2, 3, 4, 5, 8, 20))
            heads = kv_heads * rng.choice((1, 1, 2, 4, 5, 8))
            batch = _log(rng, 1, 16)
            kv = _log(rng, 16, 16000)
            q = 1 if rng.random() < 0.3 else _log(rng, 1, min(kv, 8250))
            left = _log(rng, 1, 16000)
            right = rng.choice((0, 0, 0, _log(rng, 1, 1000)))
            sinks = rng.choice((0, 4, 58, 64, rng.randint(1, 300)))
            packed = q == kv and heads == kv_heads
            case = _attention(batch, q, kv, heads, kv_heads, dim, left, right, sinks, rng.choice(("f16", "bf16")),
                              cap=kv if packed else kv + rng.randint(0, 300), q_step=rng.randint(0, max(0, q // batch)),
                              kv_step=rng.randint(0, kv // batch), lse=rng.random() < 0.5, packed=packed)
            # the scores' tensor of the plain form and the operations of the
            # largest listed case
            if heads <= 40 and batch * heads * q * case["cap"] <= 20 * 8250 * 8250 \
                    and work(case)["flops"] <= 1.6e11 and batch * case["cap"] * kv_heads * dim <= 16 * 16384 * 4 * 128:
                return case
    if op == "norm":
        while True:
            case = _norm(_log(rng, 1, 21), _log(rng, 1, 230400), rng.choice((1, 8, 16, 32)), rng.randint(1, 32),
                         rng.choice(("f16", "bf16", "f32")), act=rng.choice(("silu", "silu", "none")),
                         affine=rng.random() < 0.8, pad=rng.choice((0, 0, rng.randint(1, 64))))
            if work(case)["bytes"] <= 7.0e8:
                return case
    while True:
        rows = rng.choice((_log(rng, 1, 64), _log(rng, 1, 21658)))
        k, n = _log(rng, 64, 7680), _log(rng, 16, 15360)
        if rng.random() < 0.6:
            k, n = max(64, k // 64 * 64), max(16, n // 16 * 16)
        case = _linear(rows, k, n, rng.choice(("f16", "bf16")), act=rng.choice(("none", "silu", "gelu", "gelu_tanh")),
                       bias=rng.random() < 0.8, residual=rng.random() < 0.5, pad=rng.choice((0, 0, rng.randint(1, 64))))
        if work(case)["flops"] <= 7.67e11:
            return case


# ------------------------------------------------------------------- inputs


def lengths(case):
    """The rows and cache rows of each sequence of an attention case."""
    b = range(case["batch"])
    return ([max(0, case["q"] - case["q_step"] * i) for i in b], [max(0, case["kv"] - case["kv_step"] * i) for i in b])


def _randn(gen, shape, dtype, scale=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(scale).to(dtype)


def _padded(gen, rows, cols, pad, dtype):
    return _randn(gen, (rows, cols + pad), dtype)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "attention":
        b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:
            qkv = _randn(gen, (b, case["q"], 3, h, d), dtype)
            q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            q = _randn(gen, (b, case["q"], h, d), dtype)
            k = _randn(gen, (b, case["cap"], g, d), dtype)
            v = _randn(gen, (b, case["cap"], g, d), dtype)
        # keys grow with the head, so that some heads attend to few tokens
        # and others to many
        q.mul_(torch.linspace(0.5, 2.0, h, device="cuda", dtype=torch.float32).to(dtype)[:, None])
        q_lens, kv_lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in lengths(case))
        state.update(q=q, k=k, v=v, q_lens=q_lens, kv_lens=kv_lens,
                     out=torch.zeros((b, case["q"], h, d), dtype=dtype, device="cuda"),
                     lse=torch.zeros((b, h, case["q"]), dtype=torch.float32, device="cuda") if case["lse"] else None)
    elif case["op"] == "norm":
        c = case["groups"] * case["width"]
        x = _randn(gen, (case["frames"], case["rows"], c + case["pad"]), dtype)[:, :, :c]
        # channels with means of their own, as a convolution's bias leaves them
        x.add_(_randn(gen, (c,), dtype))
        state.update(x=x, y=torch.zeros_like(x, memory_format=torch.contiguous_format),
                     gamma=_randn(gen, (c,), torch.float32, 0.2).add_(1.0) if case["affine"] else None,
                     beta=_randn(gen, (c,), torch.float32, 0.2) if case["affine"] else None)
    else:
        m, k, n, pad = case["rows"], case["k"], case["n"], case["pad"]
        state.update(x=_padded(gen, m, k, pad, dtype), w=_randn(gen, (n, k), dtype, 1.0 / math.sqrt(k)),
                     bias=_randn(gen, (n,), torch.float32, 0.5) if case["bias"] else None,
                     residual=_padded(gen, m, n, pad, dtype) if case["residual"] else None,
                     y=torch.zeros((m, n + pad), dtype=dtype, device="cuda")[:, :n])
    return state


# ------------------------------------------------------------- plain forms


def _act(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_attention(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, n, h, d = q.shape
    g, cap = k.shape[2], k.shape[1]
    r = h // g
    qf = q.float().reshape(b, n, g, r, d).permute(0, 2, 3, 1, 4).reshape(b * g, r * n, d)
    kf = k.float().permute(0, 2, 3, 1).reshape(b * g, d, cap)
    j = torch.arange(cap, device=q.device)
    valid = j[None, :] < s["kv_lens"][:, None]
    vf = torch.where(valid[:, :, None, None], v.float(), 0.0).permute(0, 2, 1, 3).reshape(b * g, cap, d)
    i = torch.arange(n, device=q.device)
    pos = i[None, :] + (s["kv_lens"] - s["q_lens"])[:, None]
    seen = (valid[:, None, :] & (j <= pos[:, :, None] + c["right"])
            & ((j < c["sinks"]) | (j >= pos[:, :, None] - c["left"])) & (i[None, :, None] < s["q_lens"][:, None, None]))
    score = torch.matmul(qf, kf).reshape(b, g * r, n, cap).mul_(1.0 / math.sqrt(d))
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.reshape(b * g, r * n, cap), vf).reshape(b, g * r, n, d)
    out = out / torch.where(total == 0.0, 1.0, total)
    out = out.permute(0, 2, 1, 3).to(q.dtype)
    if not c["lse"]:
        return out
    lse = (top + torch.log(total))[..., 0]
    return out, torch.where(i[None, None, :] < s["q_lens"][:, None, None], lse, 0.0)


def _plain_norm(s):
    c, x = s["case"], s["x"]
    f, rows, ch = x.shape
    v = x.float().reshape(f, rows, c["groups"], c["width"])
    v = v - v.mean((1, 3), keepdim=True)
    v = (v / torch.sqrt(v.square().mean((1, 3), keepdim=True) + EPS)).reshape(f, rows, ch)
    if c["affine"]:
        v = v * s["gamma"] + s["beta"]
    return _act(v, c["act"]).to(x.dtype)


def _plain_linear(s):
    c = s["case"]
    v = torch.matmul(s["x"].float(), s["w"].float().t())
    if c["bias"]:
        v = v + s["bias"]
    v = _act(v, c["act"])
    if c["residual"]:
        v = v + s["residual"].float()
    return v.to(s["x"].dtype)


# ------------------------------------------------------- the library's own


def _library():
    path = str(Path(__file__).resolve().parent.parent / "seedvr2-ncnn-valkan_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sv2hip
    return sv2hip


def run(s):
    c = s["case"]
    if not own:
        return {"attention": _plain_attention, "norm": _plain_norm, "linear": _plain_linear}[c["op"]](s)
    lib = _library()
    if c["op"] == "attention":
        lib.sliding_attention(s["q"], s["k"], s["v"], s["out"], left=c["left"], right=c["right"], sinks=c["sinks"],
                              q_lens=s["q_lens"], kv_lens=s["kv_lens"], lse=s["lse"])
        return (s["out"], s["lse"]) if c["lse"] else s["out"]
    acts = {"none": lib.ACT_NONE, "silu": lib.ACT_SILU, "gelu": lib.ACT_GELU, "gelu_tanh": lib.ACT_GELU_TANH}
    if c["op"] == "norm":
        return lib.group_norm(s["x"], s["y"], c["groups"], gamma=s["gamma"], beta=s["beta"], eps=EPS,
                              activation=acts[c["act"]])
    return lib.linear(s["x"], s["w"], s["y"], bias=s["bias"], activation=acts[c["act"]], residual=s["residual"])


# -------------------------------------------------------------------- work


def _spans(case):
    """Of each sequence: the pairs (query, visible key) and the keys that some
    query sees."""
    for nq, nk in zip(*lengths(case)):
        pairs, seen = 0, [0, None]
        sinks = min(case["sinks"], nk)
        lowest, highest = nk, 0
        for p in range(nk - nq, nk):
            hi = min(nk, p + case["right"] + 1)
            if hi <= 0:
                continue
            lo = min(max(0, p - case["left"]), hi)
            first = min(sinks, hi, lo)
            pairs += hi - lo + first
            lowest, highest = min(lowest, lo), max(highest, hi)
        keys = max(0, highest - lowest) + min(sinks, lowest) if highest else 0
        yield nq, pairs, keys


def work(case):
    z = BYTES[case["dtype"]]
    if case["op"] == "attention":
        total_b = total_f = 0
        for nq, pairs, keys in _spans(case):
            total_b += z * case["dim"] * (2 * nq * case["heads"] + 2 * keys * case["kv_heads"])
            total_b += 4 * nq * case["heads"] if case["lse"] else 0
            total_f += 4 * pairs * case["heads"] * case["dim"]
        return {"bytes": max(1, total_b), "flops": total_f}
    if case["op"] == "norm":
        n = case["frames"] * case["rows"] * case["groups"] * case["width"]
        return {"bytes": 2 * z * n, "flops": 10 * n}
    m, k, n = case["rows"], case["k"], case["n"]
    return {"bytes": z * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + 4 * n, "flops": 2 * m * k * n}


# ------------------------------------------------------------------- exact


def _exact_attention(s):
    """Sequence by sequence and head by head, the keys of each block of
    queries gathered before the product."""
    c, d = s["case"], s["case"]["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros((c["batch"], c["heads"], c["q"]), dtype=torch.float64, device="cuda")
    share = c["heads"] // c["kv_heads"]
    for b, (nq, nk) in enumerate(zip(*lengths(c))):
        for first in range(0, nq, 1024):
            rows = torch.arange(first, min(nq, first + 1024), device="cuda")
            p = rows + (nk - nq)
            keys = torch.arange(nk, device="cuda")
            if nk:
                in_band = (keys >= int(p[0]) - c["left"]) & (keys <= int(p[-1]) + c["right"])
                keys = keys[in_band | (keys < c["sinks"])]
            hidden = ((keys[None] > p[:, None] + c["right"])
                      | ((keys[None] >= c["sinks"]) & (keys[None] < p[:, None] - c["left"])))
            empty = hidden.all(1) if keys.numel() else torch.ones_like(p, dtype=torch.bool)
            for g in range(c["kv_heads"]):
                kd, vd = s["k"][b, keys, g].double(), s["v"][b, keys, g].double()
                qd = s["q"][b, rows, g * share:(g + 1) * share].double()  # [rows, share, d]
                score = (qd.reshape(-1, d) @ kd.t()).reshape(len(rows), share, -1) / math.sqrt(d)
                score = score.masked_fill(hidden[:, None], -math.inf)
                total = torch.logsumexp(score, -1) if keys.numel() else torch.full(qd.shape[:2], -math.inf).double().cuda()
                weight = torch.where(empty[:, None, None], 0.0, torch.exp(score - total[..., None]))
                out[b, rows, g * share:(g + 1) * share] = (weight.reshape(-1, len(keys)) @ vd).reshape(len(rows), share, d)
                lse[b, g * share:(g + 1) * share, rows] = total.t()
    return (out, lse) if c["lse"] else out


def _exact_act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    if act == "gelu_tanh":
        return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "norm":
        frames = []
        for x in s["x"].double():
            v = x.reshape(case["rows"], case["groups"], case["width"]).transpose(0, 1).reshape(case["groups"], -1)
            var, mean = torch.var_mean(v, 1, unbiased=False, keepdim=True)
            v = ((v - mean) * torch.rsqrt(var + EPS)).reshape(case["groups"], case["rows"], case["width"]).transpose(0, 1)
            v = v.reshape(case["rows"], -1)
            if case["affine"]:
                v = torch.addcmul(s["beta"].double(), v, s["gamma"].double())
            frames.append(_exact_act(v, case["act"]))
        return torch.stack(frames)
    v = s["x"].double() @ s["w"].double().t()
    if case["bias"]:
        v += s["bias"].double()
    v = _exact_act(v, case["act"])
    return v + s["residual"].double() if case["residual"] else v
