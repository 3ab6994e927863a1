"""Narrow-format operators on tensors whose byte offsets pass 32 bits."""

import pytest
import torch

import ntops_amd.torch as nt

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
GIB = 1 << 30


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


def test_quantize_and_back_past_32_bits():
    n = 2 * GIB + 4096 + 64
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(4096).bfloat16().cuda()
    x[-4096:], x[:4096] = tail, tail
    codes, scales = nt.quantize_mxfp4(x)
    want = nt.quantize_mxfp4(tail)
    for part in (slice(None, 4096), slice(-4096, None)):
        c = slice(None, 2048) if part.start is None else slice(-2048, None)
        s = slice(None, 128) if part.start is None else slice(-128, None)
        assert torch.equal(codes[c], want[0]) and torch.equal(scales[s], want[1])
    assert not codes[2048:-2048].any() and not scales[128:-128].any()
    del x
    y = nt.dequantize_mxfp4(codes, scales)
    small = nt.dequantize_mxfp4(*want)
    assert torch.equal(y[:4096], small) and torch.equal(y[-4096:], small) and not y[4096:-4096].any()


@pytest.mark.parametrize("m,n,k", [(1100, 300, 512), (2100, 4000, 2048)])
def test_product_of_rows_far_apart(m, n, k):
    a, sa = nt.quantize_mxfp4(torch.randn(m, k, device="cuda"))
    b, sb = nt.quantize_mxfp4(torch.randn(n, k, device="cuda"))
    want = nt.mxfp4_mm(a, sa, b, sb)
    pitch = (5 * GIB // m) // 16 * 16
    assert m * pitch > 1 << 32
    far = torch.empty(m * pitch, dtype=torch.uint8, device="cuda").as_strided((m, a.shape[1]), (pitch, 1))
    far.copy_(a)
    assert torch.equal(nt.mxfp4_mm(far, sa, b, sb), want)


@pytest.mark.parametrize("sq", [1, 40])
@pytest.mark.parametrize("dims", [(2, 1), (1, 2)])
def test_cache_far_apart(sq, dims):
    b, h = dims
    c, d, block = 150, 64, 16
    key, value = (torch.randn(b, h, c, d, device="cuda").bfloat16() for _ in range(2))
    query = torch.randn(b, 2 * h, sq, d, device="cuda").bfloat16()

    def caches(far):
        out = []
        for _ in range(2):
            flat = torch.zeros(5 * GIB if far else b * h * c * d, dtype=torch.uint8, device="cuda")
            step = 9 * GIB // 2 if far else c * d
            out.append(flat.as_strided((b, h, c, d), (step * (h if not far else 1), step, d, 1)).view(E4M3))
        return out + [torch.ones(b, h, -(-c // block), device="cuda") for _ in range(2)]

    results = []
    for far in (False, True):
        cache = caches(far)
        nt.store_kv_cache(key, value, *cache, 0, block_size=block)
        nt.store_kv_cache(key[:, :, :3] * 100, value[:, :, :3] * 50, *cache, 130, block_size=block)
        out = nt.kv_cache_attention(query, *cache, is_causal=True, block_size=block)
        results.append([out] + [t.contiguous().float() for t in cache])
        del cache
    for x, y in zip(*results):
        assert torch.equal(x, y)
