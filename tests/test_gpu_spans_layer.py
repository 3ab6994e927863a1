"""Attention of the layers of a decoder that reads images: positions on three axes, one
layer whose tokens see a window and a few sinks, one whose sequences share the image and
the system prompt -- a prompt, then tokens one by one, eager and captured, against the
same from the 64-bit oracle's operators on the tensors that the layer itself made."""

import math

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from oracle import spans as S
from tests.test_gpu_spans import check, doubles

pytestmark = pytest.mark.gpu

B, HQ, HKV, D, WINDOW, SINKS, SECTIONS = 3, 8, 2, 128, 48, 4, (16, 24, 24)
PREFIX, CAPACITY = 150, 96


class Layer:
    """Keys and values of its own, written where each sequence ends."""

    def __init__(self, prefix):
        self.k, self.v = (torch.zeros(B, HKV, CAPACITY, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.prefix = prefix
        angles = torch.arange(4096, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
        self.sin, self.cos = angles.sin().float().cuda(), angles.cos().float().cuda()

    def __call__(self, q, k, v, positions, start, lengths):
        """q, k (batch, tokens, heads, dim); start: a tensor, where each sequence's tokens go."""
        q, k = nt.multi_axis_rotary_position_embedding_qk(q, k, self.sin, self.cos, positions, SECTIONS, interleaved=False)
        at = start[:, None, None, None] + torch.arange(k.shape[1], device="cuda")[None, None, :, None]
        at = at.expand(B, HKV, -1, D)
        self.k.scatter_(2, at, k.transpose(1, 2))
        self.v.scatter_(2, at, v.transpose(1, 2))
        q = q.transpose(1, 2)
        if self.prefix is None:
            return q, nt.sliding_window_attention(q, self.k, self.v, WINDOW, SINKS, lengths)
        return q, nt.shared_prefix_attention(q, *self.prefix, self.k, self.v, None, lengths)


def inputs(tokens):
    q, k = (torch.randn(B, tokens, h, D, device="cuda").bfloat16() for h in (HQ, HKV))
    return q, k, torch.randn(B, tokens, HKV, D, device="cuda").bfloat16()


@pytest.mark.parametrize("shared", [False, True])
def test_prompt_then_tokens(shared):
    prefix = tuple(torch.randn(1, HKV, PREFIX, D, device="cuda").bfloat16() for _ in range(2)) if shared else None
    layer, scale = Layer(prefix), 1 / math.sqrt(D)

    def verify(q, out, lengths):
        args = [doubles(t) for t in (q, layer.k, layer.v)]
        if shared:
            want = S.shared_prefix_attention(args[0], doubles(prefix[0]), doubles(prefix[1]), *args[1:], None, lengths.tolist(), scale)
        else:
            want = S.sliding_window_attention(*args, WINDOW, SINKS, lengths.tolist(), scale)
        check(out, want, CAPACITY + PREFIX, D, scale)

    tokens = 60
    lengths = torch.full((B,), tokens, device="cuda")
    at = torch.arange(tokens, device="cuda")
    grid = torch.stack((at * 0 + 5, 5 + at // 8, 5 + at % 8))[:, None].expand(3, B, tokens)
    q, k, v = inputs(tokens)
    rotated, out = layer(q, k, v, grid, torch.zeros_like(lengths), lengths)
    want = S.multi_axis_rotary_position_embedding(doubles(q), doubles(layer.sin), doubles(layer.cos), grid.cpu().numpy(), SECTIONS, False)
    assert np.abs(doubles(rotated.transpose(1, 2)) - want).max() <= 2.0**-8 * np.abs(want).max() + 1e-6
    verify(rotated, out, lengths)
    verify_tokens(layer, lengths, verify)


def verify_tokens(layer, lengths, verify):
    """Single tokens: eager ones, then a captured step replayed, beside an eager step."""
    lengths.copy_(torch.tensor([20, 60, 41]))  # sequences end where they like
    q, k, v = inputs(1)
    positions = torch.zeros(3, B, 1, dtype=torch.int64, device="cuda")
    start = torch.zeros_like(lengths)

    def step():
        return layer(q, k, v, positions, start, lengths)

    def feed(i):
        for t, x in zip((q, k, v), inputs(1)):
            t.copy_(x)
        start.copy_(lengths)
        lengths.add_(1)
        positions.copy_((lengths + 7 * i)[None, :, None].expand(3, B, 1))

    for i in range(3):
        feed(i)
        rotated, out = step()
        verify(rotated, out, lengths)
    graph = torch.cuda.CUDAGraph()
    feed(3)
    with torch.cuda.graph(graph):
        rotated, out = step()
    for i in range(4, 8):
        graph.replay()
        verify(rotated, out, lengths)
        again = step()[1]
        assert torch.equal(out, again)
        feed(i)
