"""The key / value cache in 8 bits on the GPU: store_kv_cache bit for bit and
kv_cache_attention within its roundings, against the 64-bit oracle."""

import math

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import narrow as N

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3 = torch.float8_e4m3fn


def tokens(*shape, dtype=torch.float32):
    """Normal values, a factor of their own for each channel and each token."""
    x = torch.randn(*shape) * torch.exp(torch.randn(shape[-1])) * torch.exp(torch.randn(shape[:-1]))[..., None]
    return x.clamp(-6e4, 6e4).to(dtype)


def random_cache(b, h, c, d, block, device="cuda"):
    codes = torch.randint(0, 256, (b, h, c, d), dtype=torch.uint8)
    codes[(codes & 127) == 127] = 0
    scale = torch.exp2(torch.randint(-12, 4, (b, h, -(-c // block))).float())
    return codes.view(E4M3).to(device), scale.to(device)


def doubles(t):
    return t.detach().float().cpu().double().numpy()  # (e4m3 through fp32, exactly)


def same(got, want):
    assert np.array_equal(np.nan_to_num(got, nan=-1e9), np.nan_to_num(want, nan=-1e9))


def check_store(key, value, caches, positions, lengths, block):
    """Stores in place and compares with the oracle; caches: kc, vc, ks, vs."""
    b, s = key.shape[0], key.shape[2]
    pos = [positions] * b if isinstance(positions, int) else positions.tolist()
    count = [s] * b if lengths is None else lengths.tolist()
    want = [
        N.store_kv_cache(doubles(x), doubles(c), doubles(sc), pos, count, block)
        for x, c, sc in ((key, caches[0], caches[2]), (value, caches[1], caches[3]))
    ]
    nt.store_kv_cache(key, value, *caches, positions, lengths, block_size=block)
    for i in range(2):
        same(doubles(caches[2 + i]), want[i][1])
        same(doubles(caches[i]), want[i][0])


def caches_of(b, h, c, d, block):
    (kc, ks), (vc, vs) = random_cache(b, h, c, d, block), random_cache(b, h, c, d, block)
    return [kc, vc, ks, vs]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "b,h,s,d,c,block",
    [
        (1, 1, 1, 8, 16, 16), (2, 3, 1, 128, 100, 16), (3, 2, 5, 64, 64, 32), (2, 2, 40, 80, 101, 16), (4, 1, 64, 128, 256, 64),
        (2, 2, 130, 96, 300, 64), (1, 2, 200, 128, 512, 128), (2, 1, 33, 7, 90, 16), (1, 1, 300, 36, 310, 32), (2, 1, 300, 128, 700, 512),
    ],
)
def test_store(b, h, s, d, c, block, dtype):
    caches = caches_of(b, h, c, d, block)
    key, value = (tokens(b, h, s, d, dtype=dtype).cuda() for _ in range(2))
    positions = torch.randint(0, c - s + 1, (b,), dtype=torch.int32).cuda()
    lengths = torch.randint(1, s + 1, (b,)).cuda()
    check_store(key, value, caches, positions, lengths, block)
    check_store(key, value, caches, positions, lengths, block)  # the same again changes nothing
    check_store(value, key, caches, 0, None, block)
    check_store(key, value, caches, positions.long(), None, block)


def test_numbers_past_64_bits_and_shared_caches():
    b, h, c, d = 2, 2, 50, 64
    caches = caches_of(b, h, c, d, 16)
    x = tokens(b, h, 3, d).cuda()
    before = [t.clone() for t in caches]
    for position in (1 << 70, -(1 << 70), c, -3):
        nt.store_kv_cache(x, x, *caches, position, block_size=16)
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(before, caches))
    for block in (1 << 70, 1 << 64, -(1 << 70), 1 << 25):
        with pytest.raises(RuntimeError, match="power of two"):
            nt.store_kv_cache(x, x, *caches, 0, block_size=block)
        with pytest.raises(RuntimeError, match="power of two"):
            nt.kv_cache_attention(x, *caches, block_size=block)
    with pytest.raises(TypeError):
        nt.store_kv_cache(x, x, *caches, 1.5, block_size=16)
    kc, vc, ks, vs = caches
    for shared in ((kc, kc, ks, vs), (kc, vc, ks, ks)):
        with pytest.raises(RuntimeError, match="share"):
            nt.store_kv_cache(x, x, *shared, 0, block_size=16)
    nt.kv_cache_attention(x, kc, kc, ks, ks, block_size=16)  # read only


@pytest.mark.parametrize("first", [2.0**-20, 1.0, 2.0**12])
def test_store_token_by_token(first):
    b, h, c, d, block = 2, 2, 50, 64, 16
    caches = caches_of(b, h, c, d, block)
    for t in range(40):
        size = first * 2.0 ** (t % 7 - 3) if t % 3 else first
        check_store((tokens(b, h, 1, d) * size).cuda(), tokens(b, h, 1, d).cuda(), caches, torch.tensor([t, t + 7]).cuda(), None, block)


# Blocks of more values than a wave takes: several waves share one, within what
# their registers hold and past it; the parts of a block arrive one after the other.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,c,d,block", [(2, 2, 1300, 128, 1024), (1, 3, 400, 100, 64), (1, 1, 5000, 64, 4096), (1, 2, 300, 200, 128), (1, 1, 40, 257, 16)])
def test_store_large_blocks_in_parts(b, h, c, d, block, dtype):
    caches = caches_of(b, h, c, d, block)
    at = 0
    for i, s in enumerate((c // 2, 1, 37 % c, c // 3)):
        s = min(s, c - at)
        key, value = (tokens(b, h, s, d, dtype=dtype) * 2.0 ** (3 * (i % 3) - 3) for _ in range(2))
        if i == 2:
            key[0, 0, 0, 0], value[0, h - 1, s - 1, d - 1], value[0, 0, s // 2, 3] = float("inf"), float("nan"), float("-inf")
        check_store(key.cuda(), value.cuda(), caches, at, None, block)
        at += s
    check_store(key.cuda(), value.cuda(), caches, torch.tensor([c // 4] * b).cuda(), torch.arange(1, b + 1).cuda(), block)


def test_store_drops_what_lies_outside():
    b, h, c, d, block = 6, 2, 40, 16, 16
    caches = caches_of(b, h, c, d, block)
    x = tokens(b, h, 20, d).cuda()
    big = 2**40
    check_store(x, x, caches, torch.tensor([-5, 35, 40, -20, -big, big]).cuda(), None, block)
    check_store(x, x, caches, torch.tensor([0, 3, 39, 25, 5, -19]).cuda(), torch.tensor([0, -3, 20, 99, big, -big]).cuda(), block)
    check_store(x, x, caches, -3, None, block)


def test_store_not_finite_zero_and_far():
    b, h, c, d, block = 1, 6, 32, 32, 16
    caches = caches_of(b, h, c, d, block)
    x = torch.randn(b, h, 20, d)
    x[0, 0, 3, 5], x[0, 0, 4, 6], x[0, 1, 0, 0] = float("nan"), float("inf"), float("-inf")
    x[0, 2] = 0
    x[0, 3] = 1e-41
    x[0, 4] *= 2.0**-120
    x[0, 5] = 448 * 2.0**5
    x[0, 5, 1, 1] = -448 * 2.0**5 * (1 + 2.0**-7)
    check_store(x.cuda(), x.bfloat16().float().cuda(), caches, 4, None, block)
    check_store(x.bfloat16().cuda(), x.bfloat16().cuda(), caches, 4, None, block)


def test_store_keeps_a_larger_scale_of_any_value():
    caches = caches_of(1, 1, 32, 16, 16)
    caches[2].fill_(3.0)
    caches[3].fill_(0.7)
    check_store(torch.randn(1, 1, 4, 16).cuda(), torch.randn(1, 1, 4, 16).cuda(), caches, 4, None, 16)


def test_store_strides_and_untouched_rows():
    b, h, c, d, block = 2, 4, 70, 64, 32
    wide = torch.randint(0, 100, (b, c, h, 2 * d), dtype=torch.uint8, device="cuda")
    kc, vc = (wide[..., i * d : (i + 1) * d].permute(0, 2, 1, 3).view(E4M3) for i in range(2))
    sc = torch.ones(b, 2, h, 5, device="cuda")
    caches = [kc, vc, sc[:, 0, :, :3], sc[:, 1, :, 1:4]]
    new = tokens(b, 25, h, 3 * d, dtype=torch.bfloat16).cuda()
    key, value = new[..., d : 2 * d].transpose(1, 2), new[..., 2 * d :].transpose(1, 2)
    check_store(key, value, caches, torch.tensor([10, 40], dtype=torch.int32).cuda(), None, block)
    check_store(new[..., 1 : d + 1].transpose(1, 2), new[..., ::3].transpose(1, 2), caches, 3, torch.tensor([20, 7]).cuda(), block)
    check_store(new[..., :d].transpose(1, 2)[:, :, :0], new[..., :d].transpose(1, 2)[:, :, :0], caches, 3, None, block)


# -------------------------------------------------------------- attention --


def check_attention(query, caches, lengths, causal, block, scale=None, kernel=None):
    out = nt.kv_cache_attention(query, *caches, lengths, causal, scale, block_size=block)
    if kernel is not None:
        assert kernel in _lib.last_kernel(), _lib.last_kernel()
    b, hq, sq, d = query.shape
    c = caches[0].shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    n = [c] * b if lengths is None else lengths.tolist()
    q, k, v, ks, vs = (doubles(t) for t in (query, *caches))
    want = N.kv_cache_attention(q, k, v, ks, vs, n, block, causal, scale)
    size = N.kv_cache_attention(q, k, np.abs(v), ks, vs, n, block, causal, scale)
    # a score is off by delta: fp32 sums of d products, its scaling, the
    # subtraction of the maximum and the exponential; a probability by e^delta,
    # and by half a step of bf16 where it meets the values (f16: its square, in two
    # operands); the sum of the probabilities by e^delta; the result is rounded once
    at = np.arange(c)
    top = 0.0
    for i in range(b):
        m = min(max(n[i], 0), c)
        if m == 0:
            continue
        kk = np.abs(np.nan_to_num(k[i, :, :m])) * ks[i][:, at[:m] // block][..., None]
        top = max(top, float((np.abs(q[i]).reshape(k.shape[1], -1, d) @ kk.transpose(0, 2, 1)).max()) * abs(scale))
    delta = (d + 16) * 2.0**-23 * top + 2.0**-20
    rel = 2 * math.expm1(delta) + (2.0**-16 if query.dtype == torch.float16 else 2.0**-8) + c * 2.0**-24
    bound = rel * size + HALF_STEP[query.dtype] * (np.abs(want) + rel * size) + 2.0**-140
    if query.dtype == torch.float16:
        bound = bound + 2.0**-25
    got = doubles(out)
    diff = np.abs(got - want)
    bad = ~(diff <= bound) & ~(np.isnan(want) & np.isnan(got))
    assert out.shape == query.shape and out.dtype == query.dtype
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.nanmax(diff / bound)} at {np.argwhere(bad)[:4].tolist()}"
    return out


def filled(b, h, c, d, block, dtype=torch.bfloat16):
    """A cache of normal keys and values, stored by store_kv_cache."""
    caches = caches_of(b, h, c, d, block)
    key = torch.randn(b, h, c, d) * torch.exp(0.5 * torch.randn(b, h, c, 1))
    nt.store_kv_cache(key.to(dtype).cuda(), tokens(b, h, c, d, dtype=dtype).cuda(), *caches, 0, block_size=block)
    return caches


SHAPES = [  # batch, query heads, cache heads, query rows, capacity, head dim, block
    (1, 1, 1, 1, 1, 16, 16), (2, 4, 2, 1, 50, 64, 16), (3, 8, 1, 1, 300, 128, 64), (2, 6, 2, 1, 1000, 80, 32), (1, 8, 8, 1, 700, 96, 128),
    (2, 8, 2, 4, 333, 128, 16), (1, 16, 1, 1, 2049, 64, 256), (1, 32, 2, 1, 129, 128, 64), (2, 5, 5, 3, 65, 112, 64),
    (2, 4, 2, 17, 40, 64, 16), (1, 4, 1, 33, 257, 128, 64), (2, 2, 2, 130, 130, 64, 32), (1, 8, 2, 70, 500, 96, 16), (1, 3, 3, 300, 333, 128, 64),
    (3, 12, 4, 9, 200, 16, 16), (1, 2, 1, 129, 1100, 128, 1024), (1, 6, 3, 64, 64, 48, 64),
    (2, 4, 2, 1, 60, 20, 16), (1, 2, 2, 5, 90, 256, 32), (1, 4, 2, 3, 70, 192, 64), (1, 1, 1, 2, 30, 1, 16),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,h,sq,c,d,block", SHAPES)
def test_attention(b, hq, h, sq, c, d, block, dtype, causal):
    caches = filled(b, h, c, d, block, dtype)
    query = torch.randn(b, hq, sq, d).to(dtype).cuda()
    check_attention(query, caches, None, causal, block)
    lengths = torch.randint(1, c + 1, (b,), dtype=torch.int32).cuda()
    check_attention(query, caches, lengths, causal, block, 0.3)


# 17 to 32 query rows a cache head: positions and heads in the second sixteen.
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    "b,hq,h,sq,c,d,block",
    [(2, 8, 2, 5, 333, 128, 16), (1, 32, 1, 1, 2049, 128, 64), (3, 6, 2, 9, 200, 64, 32), (66, 24, 8, 7, 130, 80, 64), (1, 17, 1, 1, 40, 16, 16),
     (2, 2, 2, 32, 31, 96, 128), (37, 16, 8, 10, 2100, 48, 64), (1, 8, 2, 8, 6000, 112, 128)],
)
def test_attention_two_sixteens(b, hq, h, sq, c, d, block, dtype, causal):
    caches = filled(b, h, c, d, block, dtype)
    query = torch.randn(b, hq, sq, d).to(dtype).cuda()
    check_attention(query, caches, None, causal, block)
    assert "kv_cache_decode" in _lib.last_kernel() and "rows32" in _lib.last_kernel(), _lib.last_kernel()
    lengths = torch.randint(0, c + 1, (b,), dtype=torch.int32)
    lengths[0] = min(sq, c) // 2
    check_attention(query, caches, lengths.cuda(), causal, block, -0.3)
    query[0, hq - 1, sq - 1, 1] = float("nan")  # stays in its row
    out = check_attention(query, caches, None, causal, block)
    assert torch.isnan(out[0, hq - 1, sq - 1]).all() and torch.isnan(out).sum() == d


# More heads than compute units: blocks of fewer waves share a unit, and only long
# caches of few more heads are split.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    "b,hq,h,sq,c,d,block,split",
    [(66, 16, 8, 1, 130, 128, 32, 1), (40, 24, 8, 2, 300, 64, 16, 1), (9, 64, 64, 1, 1030, 80, 64, 1), (37, 8, 8, 3, 2050, 16, 128, 3), (520, 2, 1, 1, 2100, 32, 64, 1)],
)
def test_attention_many_heads(b, hq, h, sq, c, d, block, split, dtype):
    caches = filled(b, h, c, d, block, dtype)
    query = torch.randn(b, hq, sq, d).to(dtype).cuda()
    lengths = torch.randint(0, c + 1, (b,), dtype=torch.int32)
    lengths[:3] = torch.tensor([0, 1, c])
    check_attention(query, caches, lengths.cuda(), True, block)
    nt.kv_cache_attention(query, *caches, lengths.cuda(), block_size=block)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert f"waves4 split{split}" in _lib.last_kernel(), _lib.last_kernel()


@pytest.mark.parametrize("b,hq,h,sq,c,d,block", SHAPES[1:18:4])
def test_attention_fp32(b, hq, h, sq, c, d, block):
    check_attention(torch.randn(b, hq, sq, d).cuda(), filled(b, h, c, d, block), None, True, block)


@pytest.mark.parametrize("sq", [1, 5, 40, 150])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths(sq, causal):
    """Lengths from none to all, past both ends, around tiles and blocks; what
    lies behind a length is NaN and never read."""
    b, hq, h, c, d, block = 12, 4, 2, 200, 64, 32
    caches = filled(b, h, c, d, block)
    n = [0, 1, 2, 31, 32, 33, 63, 64, 65, 199, 200, 5000]
    for i, m in enumerate(n):
        m = min(m, c)
        for x in caches[:2]:
            x.view(torch.uint8)[i, :, m:] = 127
        for x in caches[2:]:
            x[i, :, -(-m // block) :] = float("nan")
    query = torch.randn(b, hq, sq, d).bfloat16().cuda()
    out = check_attention(query, caches, torch.tensor(n).cuda(), causal, block)
    assert not out[0].any() and torch.isfinite(out).all()
    minus = torch.tensor([-1, -(2**40)] + n[2:]).cuda()
    out = nt.kv_cache_attention(query, *caches, minus, causal, block_size=block)
    assert not out[:2].any()


@pytest.mark.parametrize("sq", [1, 7, 100])
def test_attention_scales_far_apart(sq):
    b, hq, h, c, d, block = 2, 8, 2, 300, 128, 16
    for dtype in (torch.bfloat16, torch.float16):
        caches = filled(b, h, c, d, block)
        caches[3] *= torch.exp2(torch.randint(-30, 1, caches[3].shape).float()).cuda()  # values
        caches[2] *= (torch.rand(caches[2].shape) * 2).cuda()  # keys; no powers of two
        check_attention(torch.randn(b, hq, sq, d).to(dtype).cuda(), caches, None, False, block)


@pytest.mark.parametrize("sq", [1, 3, 60])
@pytest.mark.parametrize("scale", [0.0, -0.2, 4.0])
def test_attention_scale_argument(sq, scale):
    caches = filled(2, 2, 150, 64, 32)
    check_attention(torch.randn(2, 4, sq, 64).bfloat16().cuda(), caches, torch.tensor([150, 77]).cuda(), True, 32, scale)


@pytest.mark.parametrize("sq", [1, 50])
def test_attention_nan_stays_in_its_rows(sq):
    caches = filled(2, 2, 100, 64, 16)
    caches[0].view(torch.uint8)[0, 1, 40, 3] = 127  # a NaN key
    query = torch.randn(2, 4, sq, 64).bfloat16().cuda()
    query[1, 0, 0, 0] = float("nan")
    out = check_attention(query, caches, None, False, 16)
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all()
    assert torch.isnan(out[1, 0, 0]).all() and torch.isfinite(out[1, 1:]).all()


@pytest.mark.parametrize("sq", [1, 2, 40])
def test_attention_layouts(sq):
    b, hq, h, c, d, block = 2, 4, 2, 90, 64, 16
    caches = filled(b, h, c, d, block)
    query = torch.randn(b, sq, hq, 2 * d).bfloat16().cuda()
    q = query[..., d:].transpose(1, 2)
    want = nt.kv_cache_attention(q.contiguous(), *caches, block_size=block)
    wide = torch.full((b, c, h, 2 * d), 127, dtype=torch.uint8, device="cuda")
    views = []
    for i in range(2):
        part = wide[..., i * d : (i + 1) * d]
        part.copy_(caches[i].view(torch.uint8).transpose(1, 2))
        views.append(part.permute(0, 2, 1, 3).view(E4M3))
    sc = torch.full((b, h, 2, 9), float("nan"), device="cuda")
    for i in range(2):
        sc[:, :, i, 1:7] = caches[2 + i]
    views += [sc[:, :, 0, 1:7], sc[:, :, 1, 1:7]]
    assert torch.equal(nt.kv_cache_attention(q, *views, block_size=block), want)
    # rows that start anywhere: the kernel of one wave per row
    odd = torch.zeros(b, h, c, d + 3, dtype=torch.uint8, device="cuda")
    odd[..., 3:] = caches[0].view(torch.uint8)
    check_attention(q, [odd[..., 3:].view(E4M3), *caches[1:]], None, True, block, kernel="rows")
    check_attention(query[..., ::2].transpose(1, 2), caches, None, True, block)


def test_attention_empty():
    e = caches_of(2, 2, 0, 64, 16)
    assert not nt.kv_cache_attention(torch.randn(2, 4, 3, 64, device="cuda").half(), *e, block_size=16).any()
    caches = caches_of(2, 2, 40, 64, 16)
    assert nt.kv_cache_attention(torch.empty(2, 4, 0, 64, device="cuda"), *caches, block_size=16).shape == (2, 4, 0, 64)
    assert nt.kv_cache_attention(torch.empty(2, 0, 3, 64, device="cuda"), *caches, block_size=16).shape == (2, 0, 3, 64)


@pytest.mark.parametrize("sq", [1, 50])
def test_attention_side_stream_and_graph(sq):
    b, hq, h, c, d, block = 3, 8, 2, 900, 128, 64
    caches = filled(b, h, c, d, block)
    lengths = torch.tensor([900, 20, 400], dtype=torch.int32).cuda()
    query = torch.randn(b, hq, sq, d).bfloat16().cuda()
    want = nt.kv_cache_attention(query, *caches, lengths, True, block_size=block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nt.kv_cache_attention(query, *caches, lengths, True, block_size=block)
    side.synchronize()
    assert torch.equal(got, want)
    key, value = (torch.randn(b, h, sq, d).bfloat16().cuda() for _ in range(2))
    at = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step():
        nt.store_kv_cache(key, value, *caches, at, block_size=block)
        return nt.kv_cache_attention(query, *caches, lengths, True, block_size=block)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for t in (key, value, query):
            t.copy_(torch.randn(t.shape))
        at.copy_(torch.tensor([800 - 7 * i, 10 * i, 300]))
        lengths.copy_(torch.tensor([850 + i, 10 * i + sq, 17 * i], dtype=torch.int32))
        before = [t.clone() for t in caches]
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        after = [t.clone() for t in caches]
        for t, x in zip(caches, before):
            t.copy_(x)
        assert torch.equal(got, step())
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(after, caches))
