"""Attention over keys and queries near the ends of the range that their types hold."""

import pytest
import torch

import ntops_amd.torch as nt
from tests.test_gpu_kv_cache import caches_of, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [-111, -113])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sq", [1, 7, 90])
def test_small_keys_under_large_queries(sq, dtype, exponent):
    """Scores of size 1 of keys whose scales lie near the type's least exponents.  (A query's
    products with the codes, here up to 2^124 in sum, are fp32.)"""
    b, hq, h, c, d, block = 2, 4, 2, 300, 128, 64
    caches = caches_of(b, h, c, d, block)
    nt.store_kv_cache((torch.randn(b, h, c, d) * 2.0**exponent).cuda(), torch.randn(b, h, c, d).cuda(), *caches, 0, block_size=block)
    assert caches[2].max() <= 2.0 ** (exponent - 5)
    query = (torch.randn(b, hq, sq, d) * 2.0**-exponent).to(dtype).cuda()
    check_attention(query, caches, torch.tensor([c, c // 2]).cuda(), True, block)
