"""multi_axis_rotary_position_embedding_qk on the GPU, against the 64-bit oracle.

Tolerance, per element: the output's rounding (half a step of it, and for float16
half its least subnormal), and two products and their difference in fp32, each off by
2^-24 of its own size at most: 3 * 2^-24 (|x0 cos| + |x1 sin|)."""

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from oracle import spans as S

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def tables(rows, cols, dtype=torch.float32, pairs=None):
    rates = 1e4 ** (-torch.arange(pairs or cols, dtype=torch.float64) / (pairs or cols))
    angles = torch.arange(rows, dtype=torch.float64)[:, None] * rates
    if pairs:
        angles = angles.repeat_interleave(2, 1) + 0.1 * torch.arange(cols)
    return angles.sin().to(dtype).cuda(), angles.cos().to(dtype).cuda()


def check(x, got, sin, cos, positions, sections, interleaved):
    xd, s, c, pos = (t.detach().cpu().double().numpy() for t in (x, sin, cos, positions))
    pos = pos.astype(np.int64)
    want = S.multi_axis_rotary_position_embedding(xd, s, c, pos, sections, interleaved)
    # the same with every term positive: x0 |cos| + x1 |sin|
    size = np.abs(S.multi_axis_rotary_position_embedding(np.abs(xd), -np.abs(s), np.abs(c), pos, sections, interleaved))
    other = np.abs(S.multi_axis_rotary_position_embedding(np.abs(xd), np.abs(s), np.abs(c), pos, sections, interleaved))
    tol = HALF_STEP[x.dtype] * np.abs(want) + 3 * 2.0**-24 * np.maximum(size, other) + (2.0**-25 if x.dtype == torch.float16 else 1e-40)
    g = got.detach().cpu().double().numpy()
    assert g.shape == want.shape and np.array_equal(np.isnan(g), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(g - want)[fine] <= tol[fine]).all()


CASES = [
    # batch, seq, query heads, key heads, dim, axes, sections
    (1, 1, 1, 1, 2, 1, (1,)), (2, 1, 4, 2, 128, 3, (16, 24, 24)), (3, 7, 8, 1, 64, 3, (8, 12, 12)), (2, 33, 5, 3, 80, 2, (13, 27)),
    (1, 20, 32, 8, 128, 3, (1,) * 64), (2, 9, 3, 3, 96, 4, (10, 0, 20, 18)), (2, 5, 2, 2, 40, 3, (7, 6, 7)), (1, 6, 2, 1, 10, 2, (2, 3)),
    (2, 4, 3, 2, 512, 3, (100, 100, 56)), (1, 300, 16, 4, 128, 3, (24, 20, 20)), (2, 3, 9, 7, 128, 2, (5, 6, 7, 46)),
]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,hq,hk,d,axes,sections", CASES)
def test_rotation(b, s, hq, hk, d, axes, sections, dtype, interleaved):
    q, k = torch.randn(b, s, hq, d).to(dtype).cuda(), torch.randn(b, s, hk, d).to(dtype).cuda()
    rows = 5000
    pos = torch.randint(0, rows, (axes, b, s))
    for table, index in (
        (tables(rows, d // 2), pos.cuda()),
        (tables(rows, d // 2, dtype), pos.int().cuda()),
        (tables(rows, d, pairs=d // 2), pos[:, :1].cuda().expand(axes, b, s) if b > 1 else pos.cuda()),
        (tables(rows, d, dtype, pairs=d // 2), pos.flip(0).cuda()),
    ):
        before = q.clone(), k.clone()
        got = nt.multi_axis_rotary_position_embedding_qk(q, k, *table, index, sections, interleaved)
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
        for x, y in zip((q, k), got):
            assert y.is_contiguous()
            check(x, y, *table, index, sections, interleaved)
        assert all(torch.equal(x, y) for x, y in zip(got, nt.multi_axis_rotary_position_embedding_qk(before[0], before[1], *table, index, sections, interleaved, inplace=True)))
        assert all(torch.equal(x, y) for x, y in zip(got, before))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype, interleaved):
    b, s, hq, hk, d, sections = 2, 21, 6, 2, 64, (10, 12, 10)
    sin, cos = tables(300, d // 2)
    pos = torch.randint(0, 300, (3, b, s)).cuda()

    def forms(h):
        yield torch.randn(b, h, s, d).to(dtype).cuda().transpose(1, 2)
        yield torch.randn(b, s, h, d + 8).to(dtype).cuda()[..., 8:]
        yield torch.randn(b, s, h, d + 1).to(dtype).cuda()[..., 1:]
        yield torch.randn(b, s, d, h).to(dtype).cuda().transpose(2, 3)
        yield torch.randn(b, s, 1, d).to(dtype).cuda().expand(b, s, h, d)

    wide = torch.randn(300, d).cuda()
    for q, k in zip(forms(hq), forms(hk)):
        for table in ((sin, cos), (sin.t().contiguous().t(), cos), (wide[:, : d // 2], wide[:, d // 2 :]), (wide[:, 1 : d // 2 + 1], cos)):
            got = nt.multi_axis_rotary_position_embedding_qk(q, k, *table, pos.transpose(1, 2).contiguous().transpose(1, 2), sections, interleaved)
            for x, y in zip((q, k), got):
                check(x, y, *table, pos, sections, interleaved)
        if q.stride(2):
            q2, k2 = q.clone(memory_format=torch.preserve_format), k.clone(memory_format=torch.preserve_format)
            out = nt.multi_axis_rotary_position_embedding_qk(q2, k2, sin, cos, pos, sections, interleaved, inplace=True)
            assert out[0] is q2 and out[1] is k2
            check(q, q2, sin, cos, pos, sections, interleaved)
            check(k, k2, sin, cos, pos, sections, interleaved)
    # rows apart by a batch that is all tokens, and tables of another float type
    got = nt.multi_axis_rotary_position_embedding_qk(q, k, sin.double(), cos.double(), pos, sections, interleaved)
    for x, y in zip((q, k), got):
        check(x, y, sin, cos, pos, sections, interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
def test_positions_outside_are_nan(dtype, interleaved):
    b, s, d, sections = 2, 6, 64, (8, 12, 12)
    q, k = torch.randn(b, s, 4, d).to(dtype).cuda(), torch.randn(b, s, 2, d).to(dtype).cuda()
    sin, cos = tables(50, d // 2)
    pos = torch.randint(0, 50, (3, b, s))
    pos[0, 0, 1], pos[1, 1, 2], pos[2, 0, 5], pos[0, 1, 3] = 50, -1, 1 << 40, -(1 << 40)
    got = nt.multi_axis_rotary_position_embedding_qk(q, k, sin, cos, pos.cuda(), sections, interleaved)
    for x, y in zip((q, k), got):
        check(x, y, sin, cos, pos, sections, interleaved)
    assert torch.isnan(got[0]).sum() == 2 * 4 * (8 + 12 + 12 + 8)
    none = nt.multi_axis_rotary_position_embedding_qk(q, k, sin[:0], cos[:0], pos.cuda(), sections, interleaved)
    assert all(torch.isnan(x).all() for x in none)
    for shape in ((0, 5), (3, 0)):
        e = torch.empty(*shape, 4, d, dtype=dtype, device="cuda")
        assert nt.multi_axis_rotary_position_embedding_qk(e, e, sin, cos, torch.empty(3, *shape, dtype=torch.int64, device="cuda"), sections)[0].shape == e.shape


def test_one_axis_is_the_plain_operator():
    b, s, d = 2, 40, 128
    q, k = torch.randn(b, s, 8, d).cuda(), torch.randn(b, s, 2, d).cuda()
    sin, cos = tables(s, d // 2)
    pos = torch.arange(s).expand(3, b, s).cuda()
    for interleaved in (True, False):
        a = nt.multi_axis_rotary_position_embedding_qk(q, k, sin, cos, pos, (16, 24, 24), interleaved)
        c = nt.rotary_position_embedding_qk(q, k, sin, cos, interleaved)
        for x, y in zip(a, c):
            # both within 3 * 2^-24 of (|x0| + |x1|) of the same number
            assert (x - y).abs().max() <= 6 * 2.0**-24 * 2 * max(q.abs().max(), k.abs().max())


def test_captured_and_replayed():
    b, s, d, sections = 4, 50, 128, (16, 24, 24)
    q, k = torch.randn(b, s, 8, d).bfloat16().cuda(), torch.randn(b, s, 2, d).bfloat16().cuda()
    sin, cos = tables(900, d // 2)
    pos = torch.zeros(3, b, s, dtype=torch.int64, device="cuda")
    call = lambda: nt.multi_axis_rotary_position_embedding_qk(q, k, sin, cos, pos, sections, False)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(4):
        pos.copy_(torch.randint(0, 900, pos.shape))
        q.copy_(torch.randn(q.shape))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))
