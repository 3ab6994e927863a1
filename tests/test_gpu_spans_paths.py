"""Paths of sliding_window_attention and shared_prefix_attention that the main uses take
and small problems do not, against the 64-bit oracle (tolerances: test_gpu_spans.py)."""

import math

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from tests.test_gpu_spans import DTYPES, HALF_STEP, check, doubles, window_inputs
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


def ragged(b, c):
    """Lengths over 0 .. c, both among them."""
    return torch.randint(0, c + 1, (b,), dtype=torch.int32).index_fill_(0, torch.tensor([0]), c).index_fill_(0, torch.tensor([b - 1]), 0).cuda()


def window_twice(q, k, v, window, sinks, lengths):
    """Against the oracle, and the same bits from a second call."""
    got = nt.sliding_window_attention(q, k, v, window, sinks, lengths=lengths)
    served = _lib.last_kernel()
    scale = q.shape[3] ** -0.5
    check(got, S.sliding_window_attention(*(doubles(t) for t in (q, k, v)), window, sinks, doubles(lengths), scale), min(k.shape[2], window + sinks), q.shape[3], scale)
    again = nt.sliding_window_attention(q, k, v, window, sinks, lengths=lengths)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))
    return served


def prefix_twice(q, pk, pv, k, v, prefix_lengths, lengths):
    got = nt.shared_prefix_attention(q, pk, pv, k, v, prefix_lengths, lengths)
    served = _lib.last_kernel()
    scale = q.shape[3] ** -0.5
    want = S.shared_prefix_attention(*(doubles(t) for t in (q, pk, pv, k, v, prefix_lengths, lengths)), scale)
    check(got, want, pk.shape[2] + k.shape[2], q.shape[3], scale)
    again = nt.shared_prefix_attention(q, pk, pv, k, v, prefix_lengths, lengths)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))
    return served


# As many cache heads as a large decode batch has: a wave a block.
BATCHES = [
    # b, query heads, heads, tokens, capacity, dim, window, sinks
    (64, 8, 8, 1, 300, 128, 100, 4), (64, 16, 8, 1, 500, 64, 333, 0), (64, 16, 8, 5, 257, 128, 64, 70), (64, 32, 8, 5, 130, 64, 30, 1), (64, 32, 8, 8, 200, 96, 90, 3),
    (520, 1, 1, 1, 333, 80, 1000, 0), (513, 3, 1, 1, 90, 16, 20, 2), (128, 4, 4, 16, 100, 128, 40, 5), (72, 24, 8, 6, 150, 72, 50, 9),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hkv,sq,c,d,window,sinks", BATCHES)
def test_blocks_of_one_wave(b, hq, hkv, sq, c, d, window, sinks, dtype):
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    rows = 16 if hq // hkv * sq <= 16 else 32
    for lengths in (None, ragged(b, c)):
        assert f"waves1 rows0+{rows}" in window_twice(q, k, v, window, sinks, lengths)
        assert f"waves1 rows0+{rows}" in prefix_twice(q, k[:, :, :70], v[:, :, :70], k, v, ragged(b, 70), lengths)
    lengths = ragged(b, c).clamp(max=c - 5)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x, y = k.clone(), v.clone()
        for t in (x, y):
            t[:, :, c - 5 :, 1::3] = bad  # behind every length
        y[3, 0, 10, 2] = bad  # one value that rows may see
        window_twice(q, x, y, window, sinks, lengths)
        prefix_twice(q, k[:, :, :70], y[:, :, :70], x, y, ragged(b, 70), lengths)


# Enough rows for more than 512 blocks of 128, and with as many heads as the XCDs divide
# or not; blocks of fp32 likewise.
PROMPTS = [
    # b, query heads, heads, tokens, capacity, dim, window, sinks
    (16, 8, 8, 600, 600, 64, 200, 3), (17, 8, 8, 513, 700, 96, 1000, 0), (16, 8, 8, 520, 520, 128, 64, 1), (8, 16, 8, 600, 700, 80, 130, 40), (27, 5, 5, 600, 600, 128, 300, 7),
    (16, 8, 8, 600, 600, 192, 150, 3), (9, 24, 8, 400, 400, 136, 90, 0), (16, 8, 8, 513, 600, 256, 333, 2),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hkv,sq,c,d,window,sinks", PROMPTS)
def test_more_blocks_than_start_at_once(b, hq, hkv, sq, c, d, window, sinks, dtype):
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    assert b * hkv * -(-(hq // hkv * sq) // 128) > 512
    kernel = " f32 " if dtype == torch.float32 else " tile "
    assert kernel in window_twice(q, k, v, window, sinks, ragged(b, c))
    assert kernel in prefix_twice(q, k[:, :, :50], v[:, :, :50], k[:, :, : sq + 30], v[:, :, : sq + 30], ragged(b, 50), None)


# Prefixes attended apart, by a clear margin of what the choice goes by.
APART = [
    # groups, b, query heads, heads, tokens, prefix, capacity, dim, kernels of 16 bits and of 32
    (1, 16, 2, 2, 1, 20011, 30, 128, "few d128 waves2 rows16+16", "mode1"), (2, 32, 4, 4, 1, 9001, 9, 64, "few d64 waves2 rows16+16", "mode1"),
    (1, 40, 4, 2, 3, 6001, 50, 128, "mixed d128 rows16", "mode1"), (1, 40, 8, 2, 6, 6001, 50, 96, "mixed d96 rows32", "mode1"), (3, 96, 4, 2, 2, 5003, 21, 80, "mixed d96 rows16", "mode1"),
    (2, 60, 8, 4, 9, 6007, 33, 64, "mixed d64 rows32", "mode1"), (1, 40, 4, 2, 10, 4003, 33, 136, "tile d192 mode1", "mode1"), (1, 40, 4, 2, 3, 5003, 21, 192, "tile d192 mode1", "mode1"),
    (2, 40, 4, 2, 10, 4003, 33, 256, "tile d256 mode1", "mode1"), (1, 40, 2, 1, 7, 9001, 60, 252, None, "f32 d256 waves8 mode1"), (1, 20, 4, 2, 20, 12003, 40, 128, "tile d128 mode1", "mode1"),
]


@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d,kernel,dtype", [(*case[:8], case[9 if t == torch.float32 else 8], t) for case in APART for t in DTYPES if t == torch.float32 or case[8]])
def test_prefixes_apart(g, b, hq, hkv, sq, p, c, d, kernel, dtype):
    """The kernels by name; lengths that end inside a slice of the prefix."""
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk, pv, _ = window_inputs(g, hkv, hkv, p, p, d, dtype)
    for prefix_lengths in (None, [p - 1, 1, p // 2], [p // 3 + 17, p - 300, 0], [0, 65, p]):
        prefix_lengths = None if prefix_lengths is None else torch.tensor(prefix_lengths[:g]).cuda()
        assert kernel in prefix_twice(q, pk, pv, k, v, prefix_lengths, ragged(b, c))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d", [(1, 3, 4, 2, 1, 200, 50, 128), (2, 4, 4, 2, 40, 300, 70, 64), (1, 40, 4, 2, 3, 3001, 50, 128)])
def test_infinite_keys(g, b, hq, hkv, sq, p, c, d, dtype, bad):
    """A score of +inf leaves no number in its row, one of -inf no weight to its key."""
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk, pv, _ = window_inputs(g, hkv, hkv, p, p, d, dtype)
    pk[0, 0, p // 2, 3], k[1, 1, 0, 5] = bad, bad
    k[:, :, c - 2 :] = bad
    prefix_twice(q, pk, pv, k, v, None, torch.full((b,), c - 2).cuda())
    window_twice(q, k, v, c, 0, torch.full((b,), c - 2).cuda())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hkv,sq,c,d", [(2, 8, 2, 1, 700, 128), (1, 8, 2, 5, 500, 64), (2, 4, 2, 150, 300, 128), (1, 4, 2, 80, 300, 256), (2, 2, 1, 3, 200, 37), (64, 8, 8, 1, 200, 128), (40, 4, 2, 3, 40, 128)])
def test_scores_of_any_size(b, hq, hkv, sq, c, d, dtype):
    """Whole scores (exact in fp32) from 2^10 to 2^37, of which a row's largest, or those that
    tie for it, have all the weight."""
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    k[..., 0] = torch.randint(-90, 120, (b, hkv, c)).to(dtype).cuda()
    p = 3001 if b == 40 else 60
    pk, pv, _ = window_inputs(1, hkv, hkv, p, p, d, dtype)
    pk[..., 0] = torch.randint(-90, 121, pk.shape[:3]).to(dtype).cuda()
    for power in (10, 16, 20, 24, 26, 30):
        for sign in (1, -1):
            q.zero_()
            q[..., 0], scale = sign * 2.0 ** min(power, 15), 2.0 ** max(0, power - 15)
            args = doubles(q), doubles(k), doubles(v)
            out, size, reach = S.sliding_window_attention(*args, 90, 4, None, scale)
            check(nt.sliding_window_attention(q, k, v, 90, 4, scale=scale), (out, size, 0 * reach), 94, d, scale)
            out, size, reach = S.shared_prefix_attention(args[0], doubles(pk), doubles(pv), *args[1:], scale=scale)
            check(nt.shared_prefix_attention(q, pk, pv, k, v, scale=scale), (out, size, 0 * reach), pk.shape[2] + c, d, scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,hq,hkv,sq,c,d", [(1, 4, 2, 1, 900, 128), (2, 8, 2, 3, 200, 64), (1, 4, 2, 150, 600, 128), (1, 2, 1, 2, 300, 36), (64, 8, 8, 1, 120, 64), (2, 4, 2, 80, 400, 200)])
def test_means_of_the_largest_value(b, hq, hkv, sq, c, d, dtype):
    """All values the type's largest: so is every mean of them, though probabilities that are
    rounded up together would pass it."""
    q, k = (torch.zeros(b, h, n, d, dtype=dtype, device="cuda") for h, n in ((hq, sq), (hkv, c)))
    v = torch.full_like(k, torch.finfo(dtype).max)
    v[..., 1::2] *= -1
    q[..., 0], k[..., 1] = 1, 0
    k[:, :, 0, 0] = 1
    half = HALF_STEP[dtype]
    for p in (0.5 * (1 + 1.01 * half), 0.25 * (1 + 1.2 * half), 1 - 0.4 * half):  # every other key's probability, of a first key's 1
        scale = -math.log(p)
        want = S.sliding_window_attention(doubles(q), doubles(k), doubles(v), c, 0, None, scale)
        check(nt.sliding_window_attention(q, k, v, c, scale=scale), want, c, d, scale)
        front, own = (k[:1, :, : c // 2], v[:1, :, : c // 2]), (k[:, :, c // 2 :], v[:, :, c // 2 :])
        want = S.shared_prefix_attention(doubles(q), *(doubles(t) for t in front + own), scale=scale)
        check(nt.shared_prefix_attention(q, *front, *own, scale=scale), want, c, d, scale)
