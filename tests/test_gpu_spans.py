"""sliding_window_attention and shared_prefix_attention on the GPU, against the
64-bit oracle.

Tolerance, per element, with u the type's half step and e = 2^-24 that of fp32:
  u |o|         the output's rounding
  (u or e) a    a = softmax-weighted sum of |v|: each probability is rounded to the
                type (fp32: not at all) for the product with v
  2 ds a        a score is off by at most ds = (d + 2) e scale max_k sum |q| |k|; a
                probability, and the sum that it is divided by, by the factor e^ds
  (2 n + 16) e a  fp32 sums of n terms, of the products and of the probabilities
                (a term each at worst), and the exponentials and joins (2^-23 each)."""

import math

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import spans as S

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def values(*shape, dtype):
    """Normal values, a factor of its own for each channel."""
    return (torch.randn(*shape) * torch.exp(0.5 * torch.randn(shape[-1]))).to(dtype).cuda()


def doubles(t):
    return None if t is None else t.detach().cpu().double().numpy() if t.is_floating_point() else t.tolist()


def check(got, want, keys, d, scale):
    out, size, reach = want
    u, e = HALF_STEP[got.dtype], 2.0**-24
    ds = (d + 2) * e * abs(scale) * reach[..., None]
    tol = u * np.abs(out) + size * (max(u if got.dtype != torch.float32 else 0.0, e) + 2 * ds + (2 * keys + 16) * e) + 1e-30
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25 * (1 + size)  # below its least normal value: outputs, and probabilities (of which the largest is at least 1)
    got = doubles(got)
    assert got.shape == out.shape
    nan = np.isnan(out)
    assert np.array_equal(np.isnan(got), nan), f"{np.isnan(got).sum()} NaNs, expected {nan.sum()}"
    inf = np.isinf(out)
    assert np.array_equal(got[inf], out[inf]) and np.isfinite(got[~inf & ~nan]).all()
    fine = np.isfinite(out)
    with np.errstate(invalid="ignore"):
        over = np.abs(got[fine] - out[fine]) / tol[fine]
    assert over.size == 0 or over.max() <= 1, f"{over.max():.3g} times the tolerance"


def check_window(q, k, v, window, sinks=0, lengths=None, scale=None):
    got = nt.sliding_window_attention(q, k, v, window, sinks, lengths=lengths, scale=scale)
    s = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = S.sliding_window_attention(doubles(q), doubles(k), doubles(v), window, sinks, doubles(lengths), s)
    check(got, want, min(k.shape[2], window + sinks), q.shape[3], s)
    return got


def check_prefix(q, pk, pv, k, v, prefix_lengths=None, lengths=None, scale=None):
    got = nt.shared_prefix_attention(q, pk, pv, k, v, prefix_lengths, lengths, scale)
    s = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = S.shared_prefix_attention(*(doubles(t) for t in (q, pk, pv, k, v, prefix_lengths, lengths)), s)
    check(got, want, pk.shape[2] + k.shape[2], q.shape[3], s)
    return got


def window_inputs(b, hq, hkv, sq, c, d, dtype):
    return values(b, hq, sq, d, dtype=dtype), values(b, hkv, c, d, dtype=dtype), values(b, hkv, c, d, dtype=dtype)


def spread(b, c, dtype=torch.int32):
    """Lengths of 0, 1, the capacity and between."""
    some = [c, 0, 1, c // 2, c - 1, c // 3, 2, 3 * c // 4]
    return torch.tensor([some[i % len(some)] for i in range(b)], dtype=dtype).clamp(min=0).cuda()


WINDOWS = [
    # b, query heads, heads, tokens, capacity, dim, window, sinks
    (1, 1, 1, 1, 1, 8, 1, 0), (2, 4, 2, 1, 33, 64, 7, 2), (8, 8, 2, 1, 300, 128, 100, 4), (3, 16, 1, 1, 500, 96, 64, 1),
    (4, 32, 8, 1, 1000, 128, 333, 70), (2, 32, 1, 1, 700, 80, 129, 33), (1, 6, 2, 5, 900, 64, 200, 3), (3, 8, 1, 8, 257, 128, 31, 4),
    (2, 4, 4, 40, 100, 128, 16, 0), (8, 3, 3, 65, 65, 64, 20, 5), (2, 8, 2, 130, 400, 128, 128, 4), (1, 4, 2, 300, 300, 72, 1, 0),
    (2, 5, 5, 333, 500, 120, 64, 100), (1, 2, 1, 700, 700, 64, 255, 1), (1, 12, 3, 270, 900, 128, 1000, 10), (8, 2, 2, 17, 40, 16, 12, 3),
    (2, 2, 1, 9, 60, 200, 20, 2), (2, 3, 1, 4, 50, 37, 9, 1), (1, 2, 2, 3, 20, 256, 6, 0), (1, 1, 1, 600, 600, 128, 100, 0), (3, 4, 2, 7, 333, 128, 50, 9), (2, 16, 1, 1, 700, 92, 300, 40), (2, 4, 2, 150, 400, 256, 100, 5), (2, 2, 1, 300, 500, 160, 130, 70),
    (2, 4, 2, 150, 400, 96, 100, 5), (3, 2, 2, 333, 600, 88, 130, 70), (1, 3, 1, 700, 700, 80, 255, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,hq,hkv,sq,c,d,window,sinks", WINDOWS)
def test_window(b, hq, hkv, sq, c, d, window, sinks, dtype):
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    check_window(q, k, v, window, sinks)
    check_window(q, k, v, window, sinks, spread(b, c))
    check_window(q, k, v, window, 0, spread(b, c, torch.int64).flip(0), scale=0.3)


PREFIXES = [
    # groups, b, query heads, heads, tokens, prefix, capacity, dim
    (1, 1, 1, 1, 1, 1, 1, 8), (1, 4, 8, 2, 1, 200, 33, 64), (1, 16, 8, 2, 1, 700, 65, 128), (2, 8, 4, 4, 1, 300, 100, 96), (4, 8, 3, 3, 1, 129, 7, 64),
    (1, 30, 8, 1, 1, 1000, 20, 128), (1, 3, 8, 2, 5, 500, 64, 128), (2, 4, 16, 2, 3, 400, 31, 80), (1, 2, 4, 2, 70, 300, 70, 128),
    (1, 5, 4, 4, 100, 130, 150, 64), (3, 3, 4, 2, 40, 64, 200, 128), (1, 2, 8, 2, 150, 600, 333, 128), (1, 40, 16, 4, 4, 333, 50, 64), (2, 6, 2, 1, 7, 50, 60, 200),
    (1, 3, 3, 1, 2, 90, 5, 37), (1, 64, 32, 8, 1, 512, 10, 128), (1, 1, 8, 2, 300, 500, 300, 72),
]
# groups whose rows attend to their prefix apart from their own keys
APART = [
    (1, 16, 2, 2, 1, 10007, 30, 128), (2, 32, 4, 4, 1, 5001, 9, 64), (1, 40, 4, 2, 3, 3001, 50, 128), (2, 60, 4, 2, 10, 4003, 33, 80),
    (1, 33, 8, 8, 1, 2100, 600, 64), (1, 16, 2, 2, 33, 8001, 30, 128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d", PREFIXES + APART)
def test_prefix(g, b, hq, hkv, sq, p, c, d, dtype):
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk, pv = values(g, hkv, p, d, dtype=dtype), values(g, hkv, p, d, dtype=dtype)
    check_prefix(q, pk, pv, k, v)
    check_prefix(q, pk, pv, k, v, spread(g, p), spread(b, c))
    check_prefix(q, pk, pv, k, v, spread(g + 2, p, torch.int64)[2:], spread(b + 1, c, torch.int64)[1:], scale=0.3)


def test_a_window_past_every_key_is_causal_attention():
    q, k, v = window_inputs(2, 8, 2, 150, 400, 128, torch.bfloat16)
    whole = check_window(q, k, v, 400)
    assert torch.equal(whole, check_window(q, k, v, 1 << 70, 1 << 70))
    check_window(q, k, v, 1, 400)
    assert torch.equal(whole, check_window(q, k, v, 1 << 31, 0, torch.tensor([400, 1 << 40]).cuda()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 6, 90])
def test_lengths_outside_and_no_keys(sq, dtype):
    q, k, v = window_inputs(4, 4, 2, sq, 50, 64, dtype)
    lengths = torch.tensor([-5, 51, 1 << 40, -(1 << 40)]).cuda()
    out = check_window(q, k, v, 20, 3, lengths)
    assert not out[0].any() and not out[3].any()
    none = k[:, :, :0]
    assert not nt.sliding_window_attention(q, none, none, 5).any()
    out = check_prefix(q, k[:1], v[:1], k, v, torch.tensor([99]).cuda(), lengths)
    assert not torch.isnan(out).any()
    check_prefix(q, none[:2], none[:2], k, v, None, lengths)
    check_prefix(q, k[:2], v[:2], none, none, torch.tensor([0, 7]).cuda())
    assert not nt.shared_prefix_attention(q, none[:2], none[:2], none, none).any()
    for shape in ((0, 4, sq, 64), (4, 4, 0, 64)):
        e = torch.empty(shape, dtype=dtype, device="cuda")
        kk = torch.empty(shape[0], 2, 9, 64, dtype=dtype, device="cuda")
        assert nt.sliding_window_attention(e, kk, kk, 5).shape == shape
        assert nt.shared_prefix_attention(e, kk[:1] if shape[0] else kk, kk[:1] if shape[0] else kk, kk, kk).shape == shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,d", [(1, 128), (4, 64), (50, 128), (300, 128), (200, 64), (3, 200)])
def test_layouts(sq, d, dtype):
    """Token-major tensors, slices of wider ones, heads shared by a stride of 0, rows off
    a 16-byte boundary, last dims without a unit stride."""
    b, hq, hkv, c = 2, 4, 2, 400

    def forms(n, h):
        yield values(b, n, h, d, dtype=dtype).transpose(1, 2)
        yield values(b, h, n + 3, d + 8, dtype=dtype)[:, :, 2 : n + 2, 8:]
        yield values(b, 1, n, d, dtype=dtype).expand(b, h, n, d)
        yield values(b, h, n, d + 1, dtype=dtype)[..., 1:]
        yield values(b, h, d, n, dtype=dtype).transpose(2, 3)

    for q, k, v in zip(forms(sq, hq), forms(c, hkv), forms(c, hkv)):
        check_window(q, k, v, 90, 4, spread(b, c))
        check_prefix(q, k[:1], v[:1], k.contiguous()[:, :, :30], v[:, :, :30], torch.tensor([c - 1]).cuda())
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    check_window(q, k, k, 90)
    check_prefix(q[:1], k[:1], v[:1], k[:1], v[:1])  # a sequence that is its own prefix


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,hkv,d", [(1, 2, 128), (3, 2, 128), (7, 1, 64), (70, 2, 128), (300, 2, 64), (300, 4, 128), (9, 1, 200), (100, 2, 256), (5, 2, 38)])
def test_what_a_row_does_not_see_does_not_reach_it(sq, hkv, d, dtype, bad):
    b, hq, c, window, sinks = 2, 4, 400, 60, 3
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    lengths = torch.tensor([c - 20, c // 2]).cuda()
    places = [0, 2, sinks, 120, c // 2 - 62, c // 2 - 61, c // 2 - 30, c // 2 - 1, c // 2, c - 50, c - 21, c - 20, c - 1]
    for t, other in ((v, k), (k, v)):
        x = t.clone()
        x[:, :, places, 1::3] = bad
        args = (x, other) if t is k else (other, x)
        check_window(q, *args, window, sinks, lengths)
        # one that some rows of a block see and others do not
        x = t.clone()
        x[0, 0, c - 20 - (sq + 1) // 2, 5] = bad
        args = (x, other) if t is k else (other, x)
        check_window(q, *args, window, sinks, lengths)
        if bad != bad or t is v:
            check_prefix(q, k[:, :, :90], v[:, :, :90], *args, torch.tensor([70, 90]).cuda(), lengths)
            check_prefix(q, args[0][:1], args[1][:1], k[:, :, : sq + 5], v[:, :, : sq + 5], torch.tensor([c - 20]).cuda())
    q[0, 1, 0, 3] = bad  # a query reaches its own row
    if bad != bad:
        check_window(q, k, v, window, sinks, lengths)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d", APART)
def test_what_a_row_does_not_see_does_not_reach_it_apart(g, b, hq, hkv, sq, p, c, d, dtype, bad):
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk, pv = values(g, hkv, p, d, dtype=dtype), values(g, hkv, p, d, dtype=dtype)
    seen = [p - 37, p // 2]
    for t in (k, v):
        t[:, :, c - 3 :, 1::3] = bad
    for t in (pk, pv):
        for i in range(g):
            t[i, :, seen[i] :, ::2] = bad
    v[1, 0, c - 3 - (sq + 1) // 2, 5] = bad  # some of a sequence's rows see it
    pv[0, 0, 70, 3] = bad  # every row of a group sees it
    check_prefix(q, pk, pv, k, v, torch.tensor(seen[:g]).cuda(), torch.full((b,), c - 3).cuda())


def huge(*shape, dtype, signs):
    """Values up to the type's largest, sums of which no fp32 holds."""
    t = (torch.rand(*shape) * 0.7 + 0.25) * torch.finfo(dtype).max
    return (t * (torch.randint(0, 2, shape) * 2 - 1) if signs else t).to(dtype).cuda()


@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,hkv,d", [(1, 2, 128), (1, 4, 64), (3, 2, 128), (7, 1, 64), (70, 2, 128), (300, 2, 96), (300, 4, 128), (9, 1, 200), (5, 2, 38)])
def test_values_whose_sum_is_past_the_range(sq, hkv, d, dtype, signs):
    b, hq, c = 2, 4, 400
    q, k, _ = window_inputs(b, hq, hkv, sq, c, d, dtype)
    v = huge(b, hkv, c, d, dtype=dtype, signs=signs)
    for kk in (k, k * 0, k * 4):
        check_window(q, kk, v, 150, 3, torch.tensor([c - 20, c // 2]).cuda())
        check_prefix(q, kk[:1], v[:1], k[:, :, :90], v[:, :, :90])


@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d", APART)
def test_values_whose_sum_is_past_the_range_apart(g, b, hq, hkv, sq, p, c, d, dtype, signs):
    q, k, _ = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk = values(g, hkv, p, d, dtype=dtype)
    check_prefix(q, pk, huge(g, hkv, p, d, dtype=dtype, signs=signs), k, huge(b, hkv, c, d, dtype=dtype, signs=signs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 5, 120])
def test_scales(sq, dtype):
    q, k, v = window_inputs(2, 4, 2, sq, 300, 128, dtype)
    for scale in (0.0, -0.2, 3.0, 1e-30):
        check_window(q, k, v, 77, 2, scale=scale)
        check_prefix(q, k[:1, :, :100], v[:1, :, :100], k[:, :, :90], v[:, :, :90], scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 5, 120])
def test_scores_that_rise_and_fall(sq, dtype):
    """Keys whose scores grow along the sequence, by steps past and below what moves a
    row's reference, and the other way round."""
    q, k, v = window_inputs(1, 4, 2, sq, 600, 64, dtype)
    q = q.abs() + 0.1
    ramp = torch.linspace(0.01, 2.0, 600, device="cuda")[:, None]
    for r in (ramp, ramp.flip(0), (ramp * 20) % 2):
        kk = ((k.abs() + 0.1) * r).to(dtype)
        check_window(q, kk, v, 500, 4, scale=1.0 if dtype == torch.float32 else 0.5)
        check_prefix(q, kk, v, kk.flip(2)[:, :, : max(sq, 30)], v[:, :, : max(sq, 30)], scale=0.5)


KERNELS = [
    # tokens, query heads, heads, dim, dtype, kernel of a window, of a shared prefix of few and many keys again
    (1, 8, 2, 128, torch.bfloat16, "few", "few", "mixed"), (8, 8, 2, 64, torch.float16, "few", "few", "mixed"), (9, 8, 2, 128, torch.bfloat16, "tile", "tile", "tile"),
    (200, 8, 2, 96, torch.float16, "tile", "tile", "tile"), (3, 8, 2, 128, torch.float32, "f32", "f32", "f32"), (2, 8, 2, 100, torch.bfloat16, "rows", "rows", "rows"),
    (2, 8, 2, 98, torch.float32, "rows", "rows", "rows"), (4, 8, 2, 136, torch.float16, "tile", "tile", "tile"), (5, 8, 2, 256, torch.bfloat16, "tile", "tile", "tile"),
    (1, 4, 4, 128, torch.float32, "f32 few", "f32 few", "f32 few"), (8, 8, 4, 92, torch.float32, "f32 few", "f32 few", "f32 few"),
    (1, 4, 4, 160, torch.float32, "rows", "rows", "f32"), (9, 8, 4, 128, torch.float32, "f32 d128", "f32 d128", "f32 d128"), (5, 8, 2, 252, torch.float32, "f32", "f32", "f32"), (3, 8, 2, 250, torch.bfloat16, "rows", "rows", "rows"),
]


@pytest.mark.parametrize("sq,hq,hkv,d,dtype,window,short,long", KERNELS)
def test_kernels(sq, hq, hkv, d, dtype, window, short, long):
    """Which kernel serves a call: by rows, type and head dim; strides of a dim of one
    element do not matter."""
    q, k, v = window_inputs(4, hq, hkv, sq, 300, d, dtype)
    check_window(q, k, v, 100, 4)
    assert f" {window} " in _lib.last_kernel()
    check_prefix(q, k[:1], v[:1], k[:, :, :40], v[:, :, :40])
    nt.shared_prefix_attention(q, k[:1], v[:1], k, v)
    k1 = torch.randn(4, hkv, d, 1, device="cuda").to(dtype).transpose(2, 3)  # one token: a row stride of 1
    assert k1.stride(2) == 1
    check_window(q[:, :, :1], k1, k1, 5)
    check_prefix(q, k1[:2], k1[:2], k, v)
    check_prefix(q, k[:2], v[:2], k1, k1)
    lengthy = torch.randn(1, hkv, 20000, d, device="cuda").to(dtype)
    big = q.repeat(16, 1, 1, 1)
    kk, vv = k.repeat(16, 1, 1, 1), v.repeat(16, 1, 1, 1)
    out = nt.shared_prefix_attention(big, lengthy, lengthy, kk, vv)
    assert f" {long} " in _lib.last_kernel()
    again = nt.shared_prefix_attention(big[:4], lengthy, lengthy, kk[:4], vv[:4])
    # the same rows, joined from other slices: each within its roundings
    u = HALF_STEP[dtype] if dtype != torch.float32 else 2.0**-18
    assert ((out[:4].double() - again.double()).abs() <= 4 * u * (again.double().abs() + 1)).all()


def test_same_results_every_time():
    for sq in (1, 7, 200):
        q, k, v = window_inputs(3, 8, 2, sq, 900, 128, torch.bfloat16)
        n = spread(3, 900)
        a = [nt.sliding_window_attention(q, k, v, 400, 4, lengths=n) for _ in range(3)]
        b = [nt.shared_prefix_attention(q, k[:1], v[:1], k, v, lengths=n) for _ in range(3)]
        for x in a[1:]:
            assert torch.equal(x, a[0])
        for x in b[1:]:
            assert torch.equal(x, b[0])


@pytest.mark.parametrize("sq", [1, 5, 130])
def test_captured_and_replayed(sq):
    """Two graphs on one stream, replayed in turn with new lengths and contents, beside
    eager calls."""
    torch.manual_seed(sq)
    q, k, v = window_inputs(4, 8, 2, sq, 700, 128, torch.bfloat16)
    pk, pv = values(2, 2, 500, 128, dtype=torch.bfloat16), values(2, 2, 500, 128, dtype=torch.bfloat16)
    n, pn = spread(4, 700), spread(2, 500)
    calls = [
        lambda: nt.sliding_window_attention(q, k, v, 300, 4, lengths=n),
        lambda: nt.shared_prefix_attention(q, pk, pv, k, v, pn, n),
    ]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for f in calls:
            f()
        for f in calls:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(f())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        n.copy_(torch.randint(0, 701, (4,), dtype=torch.int32))
        pn.copy_(torch.randint(0, 501, (2,), dtype=torch.int32))
        k.copy_(values(*k.shape, dtype=k.dtype))
        for g in graphs:
            g.replay()
        want = [f() for f in calls]
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y), step


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,b,hq,hkv,sq,p,c,d", APART)
def test_captured_apart(g, b, hq, hkv, sq, p, c, d, dtype):
    """Prefixes attended apart, in a graph replayed with new lengths; twice at once, on two
    streams, beside it."""
    q, k, v = window_inputs(b, hq, hkv, sq, c, d, dtype)
    pk, pv = values(g, hkv, p, d, dtype=dtype), values(g, hkv, p, d, dtype=dtype)
    n, pn = spread(b, c), spread(g, p)

    def call():
        return nt.shared_prefix_attention(q, pk, pv, k, v, pn, n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()
        with torch.cuda.graph(graph, stream=side):
            out = call()
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        n.copy_(torch.randint(0, c + 1, (b,), dtype=torch.int32))
        pn.copy_(torch.randint(0, p + 1, (g,), dtype=torch.int32))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        want = call()
        with torch.cuda.stream(side):
            beside = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(beside, want), step


def test_on_another_stream():
    q, k, v = window_inputs(8, 8, 2, 3, 900, 128, torch.float16)
    want = nt.sliding_window_attention(q, k, v, 500, 2), nt.shared_prefix_attention(q, k[:2], v[:2], k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [(nt.sliding_window_attention(q, k, v, 500, 2), nt.shared_prefix_attention(q, k[:2], v[:2], k, v)) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for pair in got:
        assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])


def test_without_a_workspace():
    """The C entries without a workspace: the keys are not split."""
    lib = _lib.load()
    st = _lib.i64_array
    for sq in (1, 40):
        q, k, v = window_inputs(1, 8, 2, sq, 3000, 128, torch.bfloat16)
        out = torch.empty_like(q)
        args = (q.data_ptr(), st(q.stride()), k.data_ptr(), st(k.stride()), v.data_ptr(), st(v.stride()))
        assert lib.ntops_sliding_window_attention_workspace(_lib.BF16, 1, 8, 2, 1, 3000, 128, 2000, 4) > 0
        rc = lib.ntops_sliding_window_attention(
            _lib.BF16, 1, 8, 2, sq, 3000, 128, *args, None, 0, 2000, 4, 0.1, out.data_ptr(), st(out.stride()), None, 0, _lib.stream_of(q))
        assert rc == 0
        check(out, S.sliding_window_attention(doubles(q), doubles(k), doubles(v), 2000, 4, None, 0.1), 2004, 128, 0.1)
        rc = lib.ntops_shared_prefix_attention(
            _lib.BF16, 1, 1, 8, 2, sq, 3000, 3000, 128, *args, None, 0, *args[2:], None, 0, 0.1, out.data_ptr(), st(out.stride()), None, 0,
            _lib.stream_of(q))
        assert rc == 0
        check(out, S.shared_prefix_attention(doubles(q), doubles(k), doubles(v), doubles(k), doubles(v), None, None, 0.1), 6000, 128, 0.1)
