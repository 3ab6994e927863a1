"""MXFP4 products by the kernel that was measured to be the faster one for their sizes."""

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import narrow as N

pytestmark = pytest.mark.gpu


def product(m, n, k):
    a, sa = nt.quantize_mxfp4(torch.randn(m, k, device="cuda"))
    b, sb = nt.quantize_mxfp4(torch.randn(n, k, device="cuda"))
    out = nt.mxfp4_mm(a, sa, b, sb, dtype=torch.float32 if m <= 32 else torch.bfloat16)
    return [t.cpu().numpy() for t in (a, sa, b, sb)], out, _lib.last_kernel()


def on_256_units():
    return torch.cuda.get_device_properties(0).multi_processor_count == 256


@pytest.mark.parametrize("m,n,k,kernel", [(17, 6144, 4096, "j2 m32"), (32, 14336, 4096, "j2 m32"), (32, 4096, 4096, "j1 m32"), (20, 2000, 3000, "j1 m32"), (31, 66000, 64, "j2 m32")])
def test_columns_of_17_to_32_rows(m, n, k, kernel):
    operands, out, ran = product(m, n, k)
    assert not on_256_units() or kernel in ran, ran
    want = N.mxfp4_mm(*operands)
    v = [np.abs(N.dequantize_mxfp4(*operands[i : i + 2])) for i in (0, 2)]
    # fp32 sums of k exact products, in any order
    assert (np.abs(out.double().cpu().numpy() - want) <= (k + 8) * 2.0**-24 * (v[0] @ v[1].T) + 2.0**-140).all()


@pytest.mark.parametrize("m", [1, 16, 17])
def test_as_many_columns_as_are_allowed(m):
    """One row of the weight for all of them: their blocks come near the threads of a grid."""
    n = 64 * 0x7FFFFF
    a, sa = nt.quantize_mxfp4(torch.randn(m, 32, device="cuda"))
    b, sb = nt.quantize_mxfp4(torch.randn(1, 32, device="cuda"))
    want = nt.mxfp4_mm(a, sa, b, sb)
    try:
        out = nt.mxfp4_mm(a, sa, b.expand(n, -1), sb.expand(n, -1))
        assert "skinny" in _lib.last_kernel(), _lib.last_kernel()
        assert all(bool((part == want).all()) for part in out.split(1 << 26, 1))
        with pytest.raises(RuntimeError, match="too large"):
            nt.mxfp4_mm(a, sa, b.expand(n + 1, -1), sb.expand(n + 1, -1))
    finally:
        out = None
        torch.cuda.empty_cache()
