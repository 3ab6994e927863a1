"""A decoder layer's attention part on narrow formats, as a server runs it: norm,
MXFP4 projections, rotary embedding, the 8-bit cache and its attention, output
projection, residual -- a prompt at once, then token by token, eagerly and as a
captured graph.  Every operator's output is checked against the 64-bit oracle on
the inputs it had."""

import math

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from oracle import narrow as N

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, DIM, BLOCK, CAPACITY = 512, 8, 2, 64, 16, 64
E4M3 = torch.float8_e4m3fn


def doubles(t):
    return t.detach().float().cpu().double().numpy()


class Layer:
    def __init__(self, batch, dtype=torch.bfloat16):
        self.batch, self.dtype = batch, dtype
        self.norm = (1 + 0.1 * torch.randn(HIDDEN)).to(dtype).cuda()
        out = (HEADS + 2 * KV_HEADS) * DIM
        self.qkv = nt.quantize_mxfp4((torch.randn(out, HIDDEN) / HIDDEN**0.5).cuda())
        self.out = nt.quantize_mxfp4((torch.randn(HIDDEN, HEADS * DIM) / HIDDEN**0.5).cuda())
        self.cache = [torch.full((batch, KV_HEADS, CAPACITY, DIM), 127, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)]
        self.cache += [torch.full((batch, KV_HEADS, CAPACITY // BLOCK), float("nan"), device="cuda") for _ in range(2)]
        angle = torch.arange(CAPACITY)[:, None] / 10000 ** (torch.arange(DIM // 2) / (DIM // 2))
        self.sin, self.cos = angle.sin().cuda(), angle.cos().cuda()

    def step(self, x, residual, positions, lengths, sin, cos, seen=None):
        """x, residual (batch, tokens, hidden) -> the new x and residual; positions
        of the first tokens, lengths after them; `seen` collects inputs and outputs."""
        seen = {} if seen is None else seen
        b, s, _ = x.shape
        h, residual = nt.add_rms_norm(x, residual, (HIDDEN,), self.norm, 1e-6)
        h = h.view(b * s, HIDDEN)
        qkv = nt.mxfp4_mm(h, None, *self.qkv, dtype=self.dtype)
        seen["qkv"] = (h, qkv)
        q, k, v = qkv.view(b, s, -1, DIM).split((HEADS, KV_HEADS, KV_HEADS), 2)
        q, k = nt.rotary_position_embedding_qk(q, k, sin, cos, interleaved=False)
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        seen["before"] = [t.clone() for t in self.cache]
        nt.store_kv_cache(k, v, *self.cache, positions, block_size=BLOCK)
        seen["store"] = (k, v, positions, [t.clone() for t in self.cache])
        o = nt.kv_cache_attention(q, *self.cache, lengths, is_causal=True, block_size=BLOCK)
        seen["attention"] = (q, lengths, o)
        o = o.transpose(1, 2).reshape(b * s, HEADS * DIM)
        y = nt.mxfp4_mm(o, None, *self.out, dtype=self.dtype)
        seen["out"] = (o, y)
        return y.view(b, s, HIDDEN), residual


def check(layer, seen):
    half = torch.finfo(layer.dtype).eps / 2
    for name, weight in (("qkv", layer.qkv), ("out", layer.out)):
        x, y = seen[name]
        a = N.dequantize_mxfp4(*N.quantize_mxfp4(doubles(x)))
        w = N.dequantize_mxfp4(*(t.cpu().numpy() for t in weight))
        want, size = a @ w.T, np.abs(a) @ np.abs(w).T
        assert (np.abs(doubles(y) - want) <= half * np.abs(want) + 2 * (a.shape[1] + 1) * 2.0**-23 * size).all()
    k, v, positions, after = seen["store"]
    n = [k.shape[2]] * layer.batch
    for i, x in enumerate((k, v)):
        codes, scale = N.store_kv_cache(doubles(x), doubles(seen["before"][i]), doubles(seen["before"][2 + i]), positions.tolist(), n, BLOCK)
        for got, want in ((after[i], codes), (after[2 + i], scale)):
            assert np.array_equal(np.nan_to_num(doubles(got), nan=-1e9), np.nan_to_num(want, nan=-1e9))
    q, lengths, o = seen["attention"]
    args = [doubles(t) for t in (q, *after)]
    args[1:3] = [np.nan_to_num(t) for t in args[1:3]]
    want = N.kv_cache_attention(*args, lengths.tolist(), BLOCK, True, 1 / math.sqrt(DIM))
    args[2] = np.abs(args[2])
    size = N.kv_cache_attention(*args, lengths.tolist(), BLOCK, True, 1 / math.sqrt(DIM))
    # scores here stay under 2^7: fp32 sums of 64 products are within 2^-10 of them
    rel = 2 * math.expm1(2.0**-10) + 2.0**-8
    assert (np.abs(doubles(o) - want) <= rel * size + half * (np.abs(want) + rel * size)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_then_tokens(dtype):
    batch, prompt = 3, 33
    layer = Layer(batch, dtype)
    zeros = torch.zeros(batch, dtype=torch.int32, device="cuda")
    x, r = (torch.randn(batch, prompt, HIDDEN).to(dtype).cuda() for _ in range(2))
    seen = {}
    x, r = layer.step(x, r, zeros, zeros + prompt, layer.sin[:prompt], layer.cos[:prompt], seen)
    check(layer, seen)
    x, r = x[:, -1:].contiguous(), r[:, -1:].contiguous()
    for t in range(prompt, prompt + 8):
        seen = {}
        x, r = layer.step(x, r, zeros + t, zeros + t + 1, layer.sin[t : t + 1], layer.cos[t : t + 1], seen)
        check(layer, seen)
    assert torch.isfinite(x).all() and torch.isfinite(r).all()


def test_tokens_as_a_graph():
    batch = 4
    layer = Layer(batch)
    at = torch.zeros(batch, dtype=torch.int64, device="cuda")
    x, r = (torch.randn(batch, 1, HIDDEN).bfloat16().cuda() for _ in range(2))
    sin, cos = layer.sin[:1].clone(), layer.cos[:1].clone()
    start = [t.clone() for t in layer.cache]

    def step():
        return layer.step(x, r, at, at + 1, sin, cos)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    inputs = [(torch.randn(batch, 1, HIDDEN).bfloat16().cuda(), torch.randn(batch, 1, HIDDEN).bfloat16().cuda()) for _ in range(20)]

    def run(call):
        for t, s in zip(layer.cache, start):
            t.copy_(s)
        got = []
        for i, (a, b) in enumerate(inputs):
            x.copy_(a)
            r.copy_(b)
            at.fill_(i)
            sin.copy_(layer.sin[i : i + 1])
            cos.copy_(layer.cos[i : i + 1])
            y = call()
            torch.cuda.synchronize()
            got.append([t.clone() for t in y])
        return got, [t.view(torch.uint8).clone() for t in layer.cache]

    def replay():
        graph.replay()
        return out

    (want, cache), (got, cache2) = run(step), run(replay)
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert all(torch.equal(s, t) for s, t in zip(cache, cache2))
