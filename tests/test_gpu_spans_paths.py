"""Paths of sliding_window_attention and shared_prefix_attention that the main uses take
and small problems do not, against the 64-bit oracle (tolerances: test_gpu_spans.py)."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from tests.test_gpu_spans import DTYPES, check, doubles, window_inputs
from oracle import spans as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 40])
def test_query_strides_below_zero(sq, dtype):
    """The C entry with a query whose heads and tokens lie from the last one back."""
    q, k, v = window_inputs(2, 8, 2, sq, 300, 128, dtype)
    back = q.flip(0, 1, 2).contiguous()
    out = torch.empty_like(q)
    st = _lib.i64_array
    last = back.data_ptr() + (back.numel() - 128) * back.element_size()
    rc = _lib.load().ntops_sliding_window_attention(
        _lib.dtype_code(dtype), 2, 8, 2, sq, 300, 128, last, st([-s for s in q.stride()[:3]] + [1]), k.data_ptr(), st(k.stride()), v.data_ptr(), st(v.stride()),
        None, 0, 100, 4, 0.1, out.data_ptr(), st(out.stride()), None, 0, _lib.stream_of(q))
    assert rc == 0
    check(out, S.sliding_window_attention(doubles(q), doubles(k), doubles(v), 100, 4, None, 0.1), 104, 128, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sq,d", [(1, 128), (5, 64), (120, 128), (3, 37)])
def test_scales_far_below_one(sq, d, dtype):
    """Scores near fp32's largest under scales near its least, and under none at all."""
    q, k, v = window_inputs(2, 4, 2, sq, 300, d, dtype)
    q, k = (t.clamp(-4, 4) * 1e18 for t in (q, k))
    for scale in (0.0, 2e-39, -2e-39, 3e-41, 1e-36):
        args = (doubles(q), doubles(k), doubles(v))
        check(nt.sliding_window_attention(q, k, v, 77, 2, scale=scale), S.sliding_window_attention(*args, 77, 2, None, scale), 79, d, scale)
        front, own = (k[:1, :, :100], v[:1, :, :100]), (k[:, :, :130], v[:, :, :130])
        want = S.shared_prefix_attention(args[0], *(doubles(t) for t in front + own), scale=scale)
        check(nt.shared_prefix_attention(q, *front, *own, scale=scale), want, 230, d, scale)
