"""multi_axis_rotary_position_embedding_qk where a thread rotates several heads, and where
a token has more heads than 32-bit indices count."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib

pytestmark = pytest.mark.gpu


def test_heads_past_32_bits():
    """1.5e9 heads of one token (24 GB), whose count times three passes 2^31: every head is
    that of a call with one."""
    heads, d = 1_500_000_000, 8
    q, none = torch.randn(1, 1, 1, d, device="cuda").bfloat16(), torch.empty(1, 1, 0, d, dtype=torch.bfloat16, device="cuda")
    sin, cos = torch.randn(9, d // 2, device="cuda"), torch.randn(9, d // 2, device="cuda")
    pos = torch.tensor([3, 8], device="cuda").view(2, 1, 1)
    want = nt.multi_axis_rotary_position_embedding_qk(q, none, sin, cos, pos, (1, 3))[0]
    out = nt.multi_axis_rotary_position_embedding_qk(q.expand(1, 1, heads, d), none, sin, cos, pos, (1, 3))[0]
    assert "generic" in _lib.last_kernel()
    assert out.shape == (1, 1, heads, d)
    for at in range(0, heads, 1 << 27):
        assert (out[:, :, at : at + (1 << 27)] == want).all(), at
