"""The operators around the DiT blocks as a clip of many frames uses them: an
attention layer of a channels-last video whose frames arrive one at a time --
group norm with SiLU, a packed qkv product with its bias, keys and values
appended to a cache, attention over the text tokens, the last frames and the
frame itself, and the output product with bias and residual.  Every stage is
held to its float64 definition on the stage's own inputs, frame by frame, and
the captured layer to the eager one."""
from __future__ import annotations

import pytest
import torch

import clip_ops_exact as ex

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, device, dtype, pixels, heads, frames, text, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.h, self.pixels, self.window, self.text = heads, pixels, 2 * pixels, text
        c = heads * 128

        def rand(*shape, scale=1.0, dt=dtype):
            return (torch.randn(shape, generator=gen, device=device) * scale).to(dt)

        self.gamma, self.beta = rand(c, scale=0.2, dt=torch.float32) + 1, rand(c, scale=0.2, dt=torch.float32)
        self.w_qkv, self.b_qkv = rand(3 * c, c, scale=c ** -0.5), rand(3 * c, scale=0.1, dt=torch.float32)
        self.w_out, self.b_out = rand(c, c, scale=c ** -0.5), rand(c, scale=0.1, dt=torch.float32)
        self.cache = torch.full((2, 1, text + frames * pixels, heads, 128), float("nan"), dtype=dtype, device=device)
        self.cache[:, :, :text] = rand(2, 1, text, heads, 128)
        self.kv_lens = torch.zeros(1, dtype=torch.int32, device=device)
        self.y = torch.empty((1, pixels, c), dtype=dtype, device=device)
        self.qkv = torch.empty((pixels, 3 * c), dtype=dtype, device=device)
        self.att = torch.empty((1, pixels, heads, 128), dtype=dtype, device=device)
        self.out = torch.empty((pixels, c), dtype=dtype, device=device)
        self.ws = torch.empty(64 << 20, dtype=torch.uint8, device=device)

    def __call__(self, hip, x, at):
        """One frame x [1, pixels, channels] whose cache rows begin at `at`."""
        n, h = self.pixels, self.h
        hip.group_norm(x, self.y, 32, gamma=self.gamma, beta=self.beta, eps=1e-6, activation=hip.ACT_SILU, workspace=self.ws)
        hip.linear(self.y[0], self.w_qkv, self.qkv, bias=self.b_qkv)
        qkv = self.qkv.view(1, n, 3, h, 128)
        self.cache[0, :, at:at + n] = qkv[:, :, 1]
        self.cache[1, :, at:at + n] = qkv[:, :, 2]
        hip.sliding_attention(qkv[:, :, 0], self.cache[0], self.cache[1], self.att, left=self.window, right=n - 1,
                              sinks=self.text, kv_lens=self.kv_lens, workspace=self.ws)
        hip.linear(self.att.view(n, h * 128), self.w_out, self.out, bias=self.b_out, residual=x[0])
        return self.out


@pytest.mark.parametrize("dtype,pixels,heads", [(torch.float16, 60, 2), (torch.bfloat16, 480, 4), (torch.float16, 1, 2)])
def test_frames_of_a_clip(hip, device, dtype, pixels, heads):
    frames, text = 5, 58
    layer = Layer(device, dtype, pixels, heads, frames, text)
    gen = torch.Generator(device=device).manual_seed(1)
    for f in range(frames):
        x = torch.randn((1, pixels, heads * 128), generator=gen, device=device).to(dtype)
        at = text + f * pixels
        layer.kv_lens.fill_(at + pixels)
        out = layer(hip, x, at)
        torch.cuda.synchronize()
        ex.close(layer.y, *ex.group_norm(x, 32, layer.gamma, layer.beta, 1e-6, 1))
        ex.close(layer.qkv, *ex.linear(layer.y[0], layer.w_qkv, layer.b_qkv, 0, None))
        q = layer.qkv.view(1, pixels, 3, heads, 128)[:, :, 0]
        want, _, tol, _ = ex.sliding_attention(q, layer.cache[0], layer.cache[1], layer.window, pixels - 1, text,
                                               128 ** -0.5, None, layer.kv_lens)
        ex.close(layer.att, want, tol)
        ex.close(out, *ex.linear(layer.att.view(pixels, -1), layer.w_out, layer.b_out, 0, x[0]))


def test_captured_layer_follows_its_inputs(hip, device):
    pixels, heads, text = 120, 2, 10
    layer = Layer(device, torch.bfloat16, pixels, heads, 3, text)
    x = torch.randn((1, pixels, heads * 128), device=device).to(torch.bfloat16)
    layer.kv_lens.fill_(text + pixels)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        layer(hip, x, text)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            layer(hip, x, text)
    for _ in range(3):
        x.normal_()
        layer.out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = layer.out.clone()
        want = layer(hip, x, text).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_stream_that_is_not_current(hip, device):
    """`stream=`: the work and its workspaces go there."""
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.randn((2, 9000, 64), generator=gen, device=device).to(torch.bfloat16)
    w = torch.randn((64, 64), generator=gen, device=device).to(torch.bfloat16)
    q = torch.randn((1, 1, 4, 128), generator=gen, device=device).to(torch.float16)
    kv = torch.randn((1, 4000, 4, 128), generator=gen, device=device).to(torch.float16)

    def calls(**more):
        y, z, o = torch.zeros_like(x), torch.zeros_like(x[0]), torch.zeros_like(q)
        torch.cuda.synchronize()
        hip.group_norm(x, y, 8, activation=hip.ACT_GELU, **more)
        hip.linear(y[1], w, z, **more)
        hip.sliding_attention(q, kv, kv, o, left=3999, **more)
        torch.cuda.synchronize()
        return y, z, o

    want = calls()
    stream = torch.cuda.Stream()
    for _ in range(3):
        for a, b in zip(calls(stream=stream), want):
            assert torch.equal(a, b)
