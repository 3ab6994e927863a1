"""multi_axis_rotary_position_embedding_qk where a thread rotates several heads, and where
a token has more heads than 32-bit indices count."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from tests.test_gpu_rope_axes import DTYPES, check, tables

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


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,per", [(9, 7, 2), (9, 7, 3), (11, 2, 4), (1, 4, 4), (5, 3, 8), (9, 4, 8), (16, 1, 5), (0, 6, 4), (17, 0, 7)])
def test_several_heads_a_thread(hq, hk, per, dtype, interleaved, inplace):
    """Heads that a thread's share and the two in flight divide or not, shares that cross from
    the query to the key; above four a share, of pairs with axes in turn.  Some tokens
    against the oracle, all against calls of so few tokens that a thread has one head."""
    d, pack = 128, 4 if dtype == torch.float32 else 8
    packs = d // 2 // (pack // 2 if interleaved else pack)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    unit = 256 * 5 * cus  # threads that every CU holds
    b, s = 2, -(-(per * unit + unit // 3) // (2 * packs * (hq + hk)))
    sections = (1,) * (d // 2) if per > 4 else (16, 24, 24)
    q, k = (torch.randn(b, s, h, d, device="cuda").to(dtype) for h in (hq, hk))
    sin, cos = tables(700, d // 2)
    pos = torch.randint(0, 700, (3, b, s), device="cuda")
    few = max(1, unit // (2 * packs * (hq + hk)))
    want = [torch.empty_like(t) for t in (q, k)]
    for at in range(0, s, few):
        cut = slice(at, at + few)
        parts = nt.multi_axis_rotary_position_embedding_qk(q[:, cut], k[:, cut], sin, cos, pos[:, :, cut], sections, interleaved)
        assert "heads1" in _lib.last_kernel()
        for w, part in zip(want, parts):
            w[:, cut] = part
    before = q.clone(), k.clone()
    got = nt.multi_axis_rotary_position_embedding_qk(q, k, sin, cos, pos, sections, interleaved, inplace=inplace)
    assert _lib.last_kernel().endswith(f"heads{per}"), _lib.last_kernel()
    at = torch.cat((torch.arange(4), torch.randint(0, s, (20,)), torch.arange(s - 4, s))).cuda()
    for x, old, y, w in zip((q, k), before, got, want):
        assert torch.equal(y, w) and torch.equal(x, y if inplace else old)
        if x.shape[2]:
            check(old[:, at], y[:, at], sin, cos, pos[:, :, at], sections, interleaved)
