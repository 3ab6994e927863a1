"""Stores of so many blocks that eight waves for each pass the threads of a grid's
x dimension."""

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from oracle import narrow as N

pytestmark = pytest.mark.gpu


def test_store_of_2_to_the_22_blocks():
    d, block, c = 33, 16, 1 << 26
    x = torch.randn(2, 1, 1, 1, d).bfloat16()
    caches = [torch.zeros(1, 1, c, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in "kv"]
    caches += [torch.zeros(1, 1, c // block, device="cuda") for _ in "kv"]
    try:
        nt.store_kv_cache(*(t.cuda().expand(1, 1, c, d) for t in x), *caches, 0, block_size=block)
        for i in range(2):
            scale = float(N.cache_scale(np.abs(x[i].double().numpy()).max()))
            want = torch.from_numpy(N.e4m3(x[i, 0, 0].double().numpy() / scale)).float().to(torch.float8_e4m3fn)
            assert bool((caches[2 + i] == scale).all())
            codes = caches[i].view(torch.uint8)[0, 0]
            for part in codes.split(1 << 22):
                assert bool((part == want.view(torch.uint8).cuda()).all())
    finally:
        del caches
        torch.cuda.empty_cache()
