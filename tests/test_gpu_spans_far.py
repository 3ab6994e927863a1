"""Windowed and shared-prefix attention where offsets pass 32 bits: long caches, tokens
far apart, many sequences."""

import math

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib

pytestmark = pytest.mark.gpu


def reference(q, k, v):
    """Rows (heads, d) over keys (n, d), in 64 bits."""
    s = q.double() @ k.double().t() / math.sqrt(q.shape[-1])
    return torch.softmax(s, -1) @ v.double()


def close(got, want, dtype, size):
    u = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-18}[dtype]
    # the output's rounding and that of each probability, on values of at most `size`
    assert ((got.double() - want).abs() <= u * want.abs() + u * size + 1e-6).all()


@pytest.mark.parametrize("dtype,sq", [(torch.bfloat16, 1), (torch.bfloat16, 40), (torch.float32, 1)])
def test_a_window_at_the_end_of_a_long_cache(dtype, sq):
    """A token-major cache of 2^31 elements and more a sequence: the window and the sinks lie
    past what 32-bit offsets from the cache's start reach."""
    heads, d = 8, 128
    c = (1 << 31) // (heads * d) + 5000  # 4 GiB in 16 bits
    k = torch.zeros(1, c, heads, d, dtype=dtype, device="cuda")
    v = torch.zeros(1, c, heads, d, dtype=dtype, device="cuda")
    w, sinks = 700, 3
    for t in (k, v):
        t[:, : sinks + 50].normal_()
        t[:, -w - sq - 50 :].normal_()
    q = torch.randn(1, heads, sq, d, device="cuda").to(dtype)
    out = nt.sliding_window_attention(q, k.transpose(1, 2), v.transpose(1, 2), w, sinks)
    size = v.abs().max().double()
    for i in {0, sq - 1}:
        p = c - sq + i
        at = torch.cat((torch.arange(sinks), torch.arange(p - w + 1, p + 1))).cuda()
        for h in (0, heads - 1):
            close(out[0, h, i], reference(q[0, h, i : i + 1], k[0, at, h], v[0, at, h])[0], dtype, size)


def test_a_whole_cache_past_what_a_span_addresses():
    """A window over tokens that are 2 MiB apart, 2100 of them: the kernel for any layout
    serves them, and sequences past 32-bit offsets from the first."""
    d, far = 64, 1 << 20
    b = 2
    base = torch.empty(b * 2100 * far, dtype=torch.bfloat16, device="cuda")
    k = base.as_strided((b, 1, 2100, d), (2100 * far, far, far, 1))
    k.normal_()
    q = torch.randn(b, 2, 1, d, device="cuda").bfloat16()
    out = nt.sliding_window_attention(q, k, k, 5000)
    assert "rows" in _lib.last_kernel()
    for i in range(b):
        close(out[i, :, 0], reference(q[i, :, 0], k[i, 0], k[i, 0]), torch.bfloat16, k.abs().max().double())
    out = nt.shared_prefix_attention(q, k[:1, :, :2000], k[:1, :, :2000], k[:, :, :100], k[:, :, :100])
    for i in range(b):
        both = torch.cat((k[0, 0, :2000], k[i, 0, :100]))
        close(out[i, :, 0], reference(q[i, :, 0], both, both), torch.bfloat16, k.abs().max().double())


def test_many_sequences_behind_one_prefix():
    """Queries and keys of a batch past 2^31 elements."""
    b, hkv, d, c = 300, 8, 128, 7100  # 2.2e9 elements of keys
    k = torch.empty(b, hkv, c, d, dtype=torch.bfloat16, device="cuda").normal_()
    pk = torch.randn(1, hkv, 5000, d, device="cuda").bfloat16()
    q = torch.randn(b, hkv, 1, d, device="cuda").bfloat16()
    out = nt.shared_prefix_attention(q, pk, pk, k, k)
    win = nt.sliding_window_attention(q, k, k, 1000, 5)
    size = k.abs().max().double()
    for i in (0, b // 2, b - 1):
        for h in (0, hkv - 1):
            both = torch.cat((pk[0, h], k[i, h]))
            close(out[i, h, 0], reference(q[i, h], both, both)[0], torch.bfloat16, size)
            at = torch.cat((torch.arange(5), torch.arange(c - 1000, c))).cuda()
            close(win[i, h, 0], reference(q[i, h], k[i, h, at], k[i, h, at])[0], torch.bfloat16, size)
