"""What kv_cache_attention's rows make of tokens that they do not see, on every
kernel: one wave per row, the matrix cores with 16 and 32 rows a cache head, in
slices, with two blocks a compute unit, and in tiles."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn

# batch, query heads, cache heads, query rows, capacity, head dim, block, kernel
KERNELS = [
    (3, 4, 2, 8, 90, 64, 16, "rows16"), (2, 8, 2, 4, 333, 128, 64, "rows16"), (3, 8, 2, 5, 333, 128, 16, "rows32"),
    (2, 2, 2, 32, 131, 80, 64, "rows32"), (2, 8, 2, 4, 6000, 128, 64, "rows16 waves8 split"), (1, 6, 2, 9, 3000, 64, 32, "rows32 waves8 split"),
    (66, 16, 8, 2, 130, 128, 32, "rows16 waves4"), (66, 24, 8, 7, 130, 80, 64, "rows32 waves4"), (3, 4, 2, 70, 200, 128, 64, "tile d128"),
    (3, 3, 3, 150, 160, 48, 16, "tile d64"), (1, 2, 1, 129, 1100, 128, 1024, "tile d128"), (2, 4, 4, 200, 900, 64, 32, "tile d64"),
    (2, 4, 2, 5, 60, 20, 16, "attention rows"), (1, 4, 2, 9, 70, 256, 32, "attention rows"),
]


def cache(b, h, c, d, block):
    """A cache of normal keys and values that fill it."""
    key, value = (torch.randn(b, h, c, d).bfloat16().cuda() for _ in range(2))
    caches = [torch.zeros(b, h, c, d, dtype=torch.uint8, device="cuda").view(E4M3) for _ in "kv"]
    caches += [torch.zeros(b, h, -(-c // block), device="cuda") for _ in "kv"]
    nt.store_kv_cache(key, value, *caches, 0, block_size=block)
    return caches


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,h,sq,c,d,block,kernel", KERNELS)
def test_rows_that_see_nothing_are_zero(b, hq, h, sq, c, d, block, kernel, dtype):
    """Sequences shorter than their query rows, whose only tokens are NaN."""
    caches = cache(b, h, c, d, block)
    caches[1].view(torch.uint8)[:, :, : sq - 1, d // 2 :] = 127
    caches[1].view(torch.uint8)[:, :, : sq - 1, 0] = 255
    lengths = torch.tensor([(0, 1, sq // 2, sq - 1)[(i + 1) % 4] for i in range(b)], dtype=torch.int32)
    query = torch.randn(b, hq, sq, d).to(dtype).cuda()
    out = nt.kv_cache_attention(query, *caches, lengths.cuda(), True, block_size=block)
    assert kernel in _lib.last_kernel(), _lib.last_kernel()
    for i, n in enumerate(lengths.tolist()):
        assert torch.equal(out[i, :, : sq - n], torch.zeros_like(out[i, :, : sq - n]))
        assert torch.isnan(out[i, :, sq - n :, d // 2 :]).all() and torch.isnan(out[i, :, sq - n :, 0]).all()
    again = nt.kv_cache_attention(query.float(), *caches, lengths.cuda(), True, block_size=block)
    assert torch.equal(torch.isnan(out), torch.isnan(again))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,h,sq,c,d,block,kernel", KERNELS)
def test_nan_values_reach_the_rows_that_see_them(b, hq, h, sq, c, d, block, kernel, dtype, causal):
    """All else is, bit for bit, what zeros in their place give."""
    caches = cache(b, h, c, d, block)
    lengths = [(c, min(c, sq + c // 2), sq // 2 + 1, min(c, sq + 3))[i % 4] for i in range(b)]
    query = torch.randn(b, hq, sq, d).to(dtype).cuda()
    # (sequence, token, columns) of the last cache head: the last token, one that about
    # half of the rows see, and an early one
    bad = [(i, max(0, n - 1 - back), at) for i, n in enumerate(lengths) for back, at in ((0, slice(0, 1)), ((sq - 1) // 2, slice(d // 2, d // 2 + 9)), (c, slice(d - 1, d)))]
    codes = caches[1].view(torch.uint8)
    for i, t, at in bad:
        codes[i, h - 1, t, at] = 0
    n = torch.tensor(lengths).cuda()
    want = nt.kv_cache_attention(query, *caches, n, causal, block_size=block)
    assert kernel in _lib.last_kernel(), _lib.last_kernel()
    assert torch.isfinite(want).all()
    for i, t, at in bad:
        codes[i, h - 1, t, at] = 127 + 128 * (i % 2)
        first = max(0, t - lengths[i] + sq) if causal else 0
        want[i, hq - hq // h :, first:, at] = float("nan")
    out = nt.kv_cache_attention(query, *caches, n, causal, block_size=block)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.nan_to_num(), want.nan_to_num())
