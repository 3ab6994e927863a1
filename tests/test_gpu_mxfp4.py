"""MXFP4 on the GPU: quantize_mxfp4 and dequantize_mxfp4 bit for bit, mxfp4_mm
within the rounding of its sums and output, against the 64-bit oracle."""

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import narrow as N

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def spread(*shape, dtype=torch.float32):
    """Normal values, a factor of their own for each column."""
    return (torch.randn(*shape) * torch.exp(2 * torch.randn(shape[-1]))).to(dtype)


def check_codes(x):
    codes, scales = nt.quantize_mxfp4(x.cuda() if not x.is_cuda else x)
    want_codes, want_scales = N.quantize_mxfp4(x.cpu().double().numpy())
    assert codes.dtype == scales.dtype == torch.uint8
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    return codes, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "shape", [(1, 1), (1, 31), (1, 32), (1, 33), (3, 64), (7, 100), (5, 4096), (2, 3, 40), (129, 257), (64, 8), (50,), (4000, 96), (2000, 2080)]
)
def test_quantize(shape, dtype):
    check_codes(spread(*shape, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_and_saturation(dtype):
    # every multiple of 1/16 up to 8 under a largest value of 4 .. 8, so that
    # ties, values past 6 and the exponent's border all occur
    grid = torch.arange(0, 129, dtype=torch.float64) / 16
    rows = []
    for top in (4.0, 5.0, 5.9375, 6.0, 6.0625, 7.0, 7.9375):
        v = grid[grid <= top]
        v = torch.nn.functional.pad(v, (0, -len(v) % 31)).view(-1, 31)
        rows.append(torch.cat([v, torch.full((len(v), 1), -top, dtype=torch.float64)], 1))
    x = torch.cat(rows)
    for shift in (0, -9, 7):
        check_codes((x * 2.0**shift).to(dtype))


def test_quantize_far_exponents():
    for e in (-149, -140, -133, -128, -127, -126, -125, -124, 0, 120, 124, 125):
        x = torch.randn(4, 64, dtype=torch.float64).clamp(-3.9, 3.9) * 2.0**e
        check_codes(x.float())
        check_codes(x.bfloat16())
    check_codes(torch.randn(4, 64).half() * 2**-20)
    check_codes(torch.zeros(3, 96))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_not_finite(dtype):
    x = spread(6, 128, dtype=dtype)
    x[0, 3], x[1, 40], x[2, 127], x[4, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[4, 65] = float("inf")
    codes, scales = check_codes(x)
    v = nt.dequantize_mxfp4(codes, scales, dtype=dtype).cpu()
    assert torch.isnan(v[0, :32]).all() and torch.isnan(v[1, 32:64]).all() and torch.isfinite(v[3]).all()


def test_quantize_views():
    base = spread(40, 300, dtype=torch.bfloat16).cuda()
    for x in (base[:, :256], base[:, 3:259], base[::2, 8:264], base.t(), base[:, ::2], base[5:6, 7:8], base.view(4, 10, 300)[:, 2:5]):
        check_codes(x)


def test_quantize_empty():
    for shape in ((0, 64), (3, 0), (0, 0)):
        codes, scales = nt.quantize_mxfp4(torch.empty(shape, device="cuda"))
        blocks = -(-shape[1] // 32)
        assert codes.shape == (shape[0], 16 * blocks) and scales.shape == (shape[0], blocks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_every_code_and_scale(dtype):
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1)
    codes = torch.arange(16, dtype=torch.uint8)
    codes = (codes | codes.flip(0) << 4).repeat(256, 1)
    want = torch.from_numpy(N.dequantize_mxfp4(codes.numpy(), scales.numpy())).to(dtype)  # (64 -> 32 bits is exact here)
    got = nt.dequantize_mxfp4(codes.cuda(), scales.cuda(), dtype=dtype)
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=-5.0), torch.nan_to_num(want, nan=-5.0))


@pytest.mark.parametrize("size", [1, 31, 32, 33, 100, 4096, 5000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_round_trip_sizes(size, dtype):
    x = spread(37, size, dtype=dtype).cuda()
    codes, scales = nt.quantize_mxfp4(x)
    y = nt.dequantize_mxfp4(codes, scales, size, dtype=dtype)
    want = N.dequantize_mxfp4(codes.cpu().numpy(), scales.cpu().numpy(), size)
    assert y.shape == x.shape and np.array_equal(y.cpu().double().numpy(), want)
    # codes and scales that are views of wider tensors
    wide_c = torch.zeros(37, codes.shape[1] + 7, dtype=torch.uint8, device="cuda")
    wide_s = torch.zeros(37, scales.shape[1] + 3, dtype=torch.uint8, device="cuda")
    wide_c[:, 5 : 5 + codes.shape[1]], wide_s[:, 2 : 2 + scales.shape[1]] = codes, scales
    z = nt.dequantize_mxfp4(wide_c[:, 5 : 5 + codes.shape[1]], wide_s[:, 2 : 2 + scales.shape[1]], size, dtype=dtype)
    assert torch.equal(y, z)


# ---------------------------------------------------------------- product --


def check_product(a, sa, b, sb, bias, dtype):
    out = nt.mxfp4_mm(a, sa, b, sb, bias, dtype=dtype)
    m, n, k = a.shape[0], b.shape[0], 32 * sb.shape[1]
    assert out.shape == (m, n) and out.dtype == dtype
    va, vb = (N.dequantize_mxfp4(c.cpu().numpy(), s.cpu().numpy()) for c, s in ((a, sa), (b, sb)))
    want = va @ vb.T
    size = np.abs(va) @ np.abs(vb).T
    if bias is not None:
        want = want + bias.cpu().double().numpy()
        size = size + np.abs(bias.cpu().double().numpy())
    # products are exact; each of at most k + 1 fp32 additions rounds by half a
    # step of a partial sum, none of which passes the sum of magnitudes (the
    # matrix instruction adds 128 products: a full step is allowed for each),
    # then the output is rounded once
    bound = (k + 1) * 2.0**-23 * size + HALF_STEP[dtype] * (np.abs(want) + (k + 1) * 2.0**-23 * size) + 2.0**-149
    if dtype == torch.float16:
        bound = bound + 2.0**-25
    diff = np.abs(out.cpu().double().numpy() - want)
    bad = ~(diff <= bound) & ~(np.isnan(want) & out.isnan().cpu().numpy())
    assert not bad.any(), f"{bad.sum()} of {bad.size} past the bound, worst {np.nanmax(diff / bound)} at {np.argwhere(bad)[:5].tolist()}"
    return out


def operands(m, n, k, dtype=torch.float32):
    a, sa = nt.quantize_mxfp4(spread(m, k, dtype=dtype).cuda())
    b, sb = nt.quantize_mxfp4((torch.randn(n, k) / k**0.5).to(dtype).cuda())
    return a, sa, b, sb


SIZES = [
    (1, 1, 1), (1, 1, 32), (1, 16, 33), (2, 17, 256), (5, 100, 300), (16, 64, 1024), (17, 33, 96), (1, 4096, 768),
    (4, 1000, 4096), (8, 515, 2080), (16, 256, 8192), (33, 129, 512), (64, 300, 1600), (100, 1001, 2080), (128, 128, 256),
    (17, 4100, 2080), (32, 300, 4096), (25, 20000, 1030), (31, 1, 64), (32, 5000, 8200), (20, 70001, 96),
    (129, 257, 288), (200, 640, 4096), (256, 512, 1024), (300, 1000, 544), (512, 512, 2048), (1000, 777, 1056),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, dtype):
    bias = torch.randn(n).to(dtype).cuda() if (m + n) % 2 else None
    check_product(*operands(m, n, k), bias, dtype)


# Each tile in a round and in more, whole and in slices of K, scales in dwords and not.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    "m,n,k,kernel",
    [(130, 6100, 7424, "tile128 split2 stages4"), (130, 6100, 7200, "tile128 split2 stages4"), (200, 12300, 1056, "tile128 split1 stages4"),
     (300, 8300, 768, "tile128 split1 stages2"), (300, 12000, 2048, "tile128 split1 stages2"), (300, 12001, 2080, "tile128 split1 stages2"),
     (120, 40000, 256, "tile128 split1 stages2"), (64, 300, 4096, "tile64 split2 stages4"), (70, 302, 4128, "tile64 split2 stages4"),
     (40, 33000, 544, "tile64 split1 stages2"), (50, 33000, 1536, "tile64 split1 stages2"), (50, 33000, 1600, "tile64 split1 stages2"), (300, 1000, 544, "tile64 split1 stages2")],
)
def test_product_tiles(m, n, k, kernel, dtype):
    bias = torch.randn(n).to(dtype).cuda() if m % 3 else None
    args = operands(m, n, k)
    out = check_product(*args, bias, dtype)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert kernel in _lib.last_kernel(), _lib.last_kernel()
    for _ in range(3):
        assert torch.equal(nt.mxfp4_mm(*args, bias, dtype=dtype), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(2048, 4096, 1280), (2000, 4090, 1792), (1900, 4099, 2048), (2300, 7700, 1536), (8200, 4100, 1312), (2100, 4200, 1100), (2050, 4097, 1024), (2048, 8192, 1280), (2000, 8190, 1792), (1900, 8199, 2048), (1500, 2900, 8192), (1500, 5700, 7680)])
def test_product_large(m, n, k, dtype):
    bias = torch.randn(n).to(dtype).cuda() if n % 4 else None
    args = operands(m, n, k)
    out = check_product(*args, bias, dtype)
    if -(-m // 128) * -(-n // 128) > 512 and k > 1024:
        assert _lib.last_kernel() == "mxfp4_large"
    for _ in range(3):
        assert torch.equal(nt.mxfp4_mm(*args, bias, dtype=dtype), out)
    a, sa, b, sb = args
    wide = torch.full((m, sa.shape[1] + 9), 255, dtype=torch.uint8, device="cuda")
    wide[:, 3:-6] = sa
    assert torch.equal(nt.mxfp4_mm(a, wide[:, 3:-6], b, sb, bias, dtype=dtype), out)


@pytest.mark.parametrize("m,n,k", [(3, 50, 4096), (64, 200, 512), (260, 300, 1056)])
def test_product_is_the_same_every_time(m, n, k):
    args = operands(m, n, k)
    first = nt.mxfp4_mm(*args)
    for _ in range(3):
        assert torch.equal(nt.mxfp4_mm(*args), first)


@pytest.mark.parametrize("m,n,k", [(1, 96, 512), (40, 130, 1024), (300, 300, 2048)])
def test_product_of_views(m, n, k):
    a, sa, b, sb = operands(m, n, k)
    want = nt.mxfp4_mm(a, sa, b, sb, dtype=torch.float32)

    def view(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), 255, dtype=torch.uint8, device="cuda")
        wide[:, left : left + t.shape[1]] = t
        return wide[:, left : left + t.shape[1]]

    for cl, cr, sl, sr in ((0, 16, 0, 4), (16, 16, 4, 4), (1, 0, 1, 0), (3, 5, 2, 7), (0, 0, 0, 1)):
        got = nt.mxfp4_mm(view(a, cl, cr), view(sa, sl, sr), view(b, cl, cr), view(sb, sl, sr), dtype=torch.float32)
        assert torch.equal(got, want), (cl, cr, sl, sr)
    got = nt.mxfp4_mm(a.t().contiguous().t(), sa.t().contiguous().t(), b, sb, dtype=torch.float32)
    assert torch.equal(got, want)


def test_product_of_activations():
    for dtype in DTYPES:
        x = spread(9, 1000, dtype=dtype).cuda()
        b, sb = nt.quantize_mxfp4(torch.randn(70, 1000).cuda())
        assert torch.equal(nt.mxfp4_mm(x, None, b, sb), nt.mxfp4_mm(*nt.quantize_mxfp4(x), b, sb))


# Up to 4 rows of 16 bits on 16-byte addresses are rounded inside the product's
# kernel: the same codes, so the same sums, bit for bit.  One column group of a block,
# two and four; last blocks and steps that the row fills in part or not at all.
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("n,k", [(70, 8), (1, 32), (33, 1000), (200, 1024), (40, 4096 + 40), (5000, 264), (20000, 2056), (130, 4104)])
def test_product_of_few_activations(m, n, k):
    b, sb = nt.quantize_mxfp4(torch.randn(n, k).cuda())
    for dtype in DTYPES:
        x = spread(m, k, dtype=dtype).cuda()
        if n == 33:
            x[0, -1], x[m - 1, 40] = float("nan"), float("-inf")
        bias = torch.randn(n).to(dtype).cuda() if n % 3 else None
        want = nt.mxfp4_mm(*nt.quantize_mxfp4(x), b, sb, bias, dtype=dtype)
        fused = m <= 4 and dtype != torch.float32
        wide = torch.full((m, k + 24), float("nan"), dtype=dtype, device="cuda")
        for left in (8, 3, 0, None):  # on 16-byte addresses and off them, between values that are not numbers
            view = x
            if left is not None:
                view = wide.fill_(float("nan"))[:, left : left + k]
                view.copy_(x)
            got = nt.mxfp4_mm(view, None, b, sb, bias, dtype=dtype)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0)), (dtype, left)
            assert ("fused" in _lib.last_kernel()) == (fused and left != 3), (dtype, left, _lib.last_kernel())


def test_product_of_few_activations_graph_and_stream():
    b, sb = nt.quantize_mxfp4(torch.randn(640, 2048).cuda())
    x = torch.randn(3, 2048, device="cuda").half()
    want = nt.mxfp4_mm(x, None, b, sb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nt.mxfp4_mm(x, None, b, sb)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nt.mxfp4_mm(x, None, b, sb)
    for _ in range(3):
        x.copy_(torch.randn(3, 2048))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nt.mxfp4_mm(*nt.quantize_mxfp4(x), b, sb))


@pytest.mark.parametrize("m", [2, 40, 200])
def test_product_keeps_nan_blocks_apart(m):
    x, w = torch.randn(m, 512), torch.randn(60, 512)
    x[1, 100], w[7, 300] = float("nan"), float("inf")
    out = nt.mxfp4_mm(*nt.quantize_mxfp4(x.cuda()), *nt.quantize_mxfp4(w.cuda()))
    nan = torch.isnan(out).cpu()
    want = torch.zeros(m, 60, dtype=torch.bool)
    want[1], want[:, 7] = True, True
    assert torch.equal(nan, want)


def test_product_empty():
    e = lambda *s: torch.empty(s, dtype=torch.uint8, device="cuda")
    assert nt.mxfp4_mm(e(0, 64), e(0, 4), e(5, 64), e(5, 4)).shape == (0, 5)
    assert nt.mxfp4_mm(e(3, 64), e(3, 4), e(0, 64), e(0, 4)).shape == (3, 0)
    f = lambda *s: torch.empty(s, device="cuda").bfloat16()
    assert nt.mxfp4_mm(f(0, 64), None, e(5, 32), e(5, 2)).shape == (0, 5) and nt.mxfp4_mm(f(3, 64), None, e(0, 32), e(0, 2)).shape == (3, 0)
    bias = torch.randn(5, device="cuda").bfloat16()
    assert torch.equal(nt.mxfp4_mm(f(3, 0), None, e(5, 0), e(5, 0), bias), bias.expand(3, 5))
    assert torch.equal(nt.mxfp4_mm(e(3, 0), e(3, 0), e(5, 0), e(5, 0), bias), bias.expand(3, 5))


def test_product_side_stream_and_graph():
    a, sa, b, sb = operands(24, 640, 2048)
    want = nt.mxfp4_mm(a, sa, b, sb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = nt.mxfp4_mm(a, sa, b, sb)
    side.synchronize()
    assert torch.equal(got, want)
    x = torch.randn(24, 2048, device="cuda").bfloat16()
    nt.mxfp4_mm(x, None, b, sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nt.mxfp4_mm(x, None, b, sb)
    for _ in range(4):
        x.copy_(torch.randn(24, 2048))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nt.mxfp4_mm(x, None, b, sb))
