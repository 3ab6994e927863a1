"""What the windowed and shared-prefix attention and the multi-axis rotary positions
refuse, before anything is launched, and the oracle's own identities."""

import ctypes

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import spans as S


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def window(q=(2, 4, 3, 8), k=(2, 2, 10, 8), v=None, window=5, sinks=1, dtypes=(torch.float32,) * 3, **kw):
    v = k if v is None else v
    return nt.sliding_window_attention(*(zeros(*s, dtype=t) for s, t in zip((q, k, v), dtypes)), window, sinks, **kw)


def prefix(q=(4, 4, 3, 8), pk=(2, 2, 10, 8), pv=None, k=(4, 2, 7, 8), dtype=torch.float32, **kw):
    pv = pk if pv is None else pv
    return nt.shared_prefix_attention(zeros(*q), zeros(*pk, dtype=dtype), zeros(*pv, dtype=dtype), zeros(*k), zeros(*k), **kw)


def test_attention_refusals():
    for call, match in [
        (lambda: window(q=(2, 3, 8)), "4-D"),
        (lambda: window(v=(2, 2, 11, 8)), "4-D"),
        (lambda: window(q=(3, 4, 3, 8)), "does not fit"),
        (lambda: window(q=(2, 4, 3, 16)), "does not fit"),
        (lambda: window(q=(2, 3, 3, 8)), "multiple"),
        (lambda: window(k=(2, 0, 10, 8)), "multiple"),
        (lambda: window(window=0), "at least 1"),
        (lambda: window(window=-(1 << 70)), "at least 1"),
        (lambda: window(sinks=-1), "at least 0"),
        (lambda: window(dtypes=(torch.float32, torch.float16, torch.float16)), "expected one of"),
        (lambda: window(dtypes=(torch.float64,) * 3), "expected one of"),
        (lambda: window(lengths=zeros(3, dtype=torch.int32)), "lengths"),
        (lambda: window(lengths=zeros(2)), "lengths"),
        (lambda: window(), "GPU tensor"),
        (lambda: prefix(pk=(2, 10, 8)), "do not fit"),
        (lambda: prefix(pk=(2, 4, 10, 8)), "do not fit"),
        (lambda: prefix(pk=(2, 2, 10, 16)), "do not fit"),
        (lambda: prefix(pv=(2, 2, 9, 8)), "do not fit"),
        (lambda: prefix(pk=(3, 2, 10, 8)), "multiple of 3"),
        (lambda: prefix(pk=(0, 2, 10, 8)), "multiple of 0"),
        (lambda: prefix(dtype=torch.bfloat16), "expected prefixes"),
        (lambda: prefix(prefix_lengths=zeros(4, dtype=torch.int64)), "prefix_lengths"),
        (lambda: prefix(lengths=zeros(2, dtype=torch.int64)), "lengths"),
        (lambda: prefix(), "GPU tensor"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
    for bad in (2.5, "3", None):
        with pytest.raises(TypeError):
            window(window=bad)


def rope(q=(2, 5, 4, 8), k=(2, 5, 2, 8), table=(9, 4), cos=None, pos=(3, 2, 5), sections=(1, 1, 2), dtype=torch.float32, pos_dtype=torch.int64, **kw):
    return nt.multi_axis_rotary_position_embedding_qk(
        zeros(*q, dtype=dtype), zeros(*k), zeros(*table), zeros(*(cos or table)), zeros(*pos, dtype=pos_dtype), sections, **kw)


def test_rotary_refusals():
    for call, match in [
        (lambda: rope(q=(2, 5, 8)), "batch, seq, heads, dim"),
        (lambda: rope(k=(2, 4, 2, 8)), "differ"),
        (lambda: rope(dtype=torch.float16), "expected one of"),
        (lambda: rope(q=(2, 5, 4, 7), k=(2, 5, 4, 7)), "even"),
        (lambda: rope(pos=(3, 2, 4)), "positions"),
        (lambda: rope(pos=(0, 2, 5)), "positions"),
        (lambda: rope(pos_dtype=torch.float32), "positions"),
        (lambda: rope(sections=(1, 1, 1)), "add up"),
        (lambda: rope(sections=(5, -1)), "add up"),
        (lambda: rope(sections=()), "add up"),
        (lambda: rope(table=(9, 5)), "tables"),
        (lambda: rope(cos=(8, 4)), "tables"),
        (lambda: rope(), "GPU tensor"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
    q = zeros(2, 5, 1, 8).expand(2, 5, 4, 8)
    with pytest.raises(RuntimeError, match="share memory"):
        nt.multi_axis_rotary_position_embedding_qk(q, zeros(2, 5, 2, 8), zeros(9, 4), zeros(9, 4), zeros(3, 2, 5, dtype=torch.int64), (1, 1, 2), inplace=True)
    one = zeros(2, 5, 4, 8)
    with pytest.raises(RuntimeError, match="twice"):
        nt.multi_axis_rotary_position_embedding_qk(one, one, zeros(9, 4), zeros(9, 4), zeros(3, 2, 5, dtype=torch.int64), (1, 1, 2), inplace=True)
    with pytest.raises(TypeError):
        rope(sections=(1.5, 2.5))


def test_rotary_in_place_refuses_heads_of_both():
    rest = (zeros(9, 4), zeros(9, 4), zeros(3, 2, 5, dtype=torch.int64), (1, 1, 2))
    both = zeros(2, 5, 7, 8)
    for q, k in ((both[:, :, :5], both[:, :, 4:]), (both[:, :, 3:], both[:, :, :4]), (both, both[:, :, 2:3]), (both[:, :, :2], both[:, :, :1])):
        with pytest.raises(RuntimeError, match="twice"):
            nt.multi_axis_rotary_position_embedding_qk(q, k, *rest, inplace=True)
        with pytest.raises(RuntimeError, match="GPU tensor"):
            nt.multi_axis_rotary_position_embedding_qk(q, k, *rest)
    for q, k in ((both[:, :, :5], both[:, :, 5:]), (both[:, :, 4:], both[:, :, :4]), (both[:, :, :3], both.clone()[:, :, :3])):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            nt.multi_axis_rotary_position_embedding_qk(q, k, *rest, inplace=True)


def _err():
    return _lib.load().ntops_last_error().decode()


def test_c_entries_refuse():
    lib, p, st = _lib.load(), ctypes.c_void_p(256), _lib.i64_array((8, 8, 8, 1))

    def win(dtype=_lib.BF16, b=2, hq=4, hkv=2, sq=3, c=10, d=8, q=p, k=p, lengths=None, ldt=0, w=5, s=1, ws=None, nws=0):
        return lib.ntops_sliding_window_attention(dtype, b, hq, hkv, sq, c, d, q, st, k, st, k, st, lengths, ldt, w, s, 1.0, p, st, ws, nws, None)

    def pre(g=1, b=2, hq=4, hkv=2, sq=3, pl=4, c=10, d=8, pk=p, plen=None, pdt=0):
        return lib.ntops_shared_prefix_attention(_lib.F16, g, b, hq, hkv, sq, pl, c, d, p, st, pk, st, pk, st, plen, pdt, p, st, p, st, None, 0, 1.0, p, st, None, 0, None)

    for rc, code, text in [
        (win(b=-1), 1, "negative"), (win(dtype=_lib.F64), 2, "dtype"), (win(hkv=3), 1, "multiple"), (win(hkv=0), 1, "multiple"),
        (win(q=None), 1, "null"), (win(k=None), 1, "null"), (win(d=257), 2, "head dim"), (win(w=0), 1, "window"), (win(s=-1), 1, "sinks"),
        (win(lengths=p, ldt=_lib.F32), 1, "lengths"), (win(b=1 << 40), 2, "too large"), (win(c=1 << 31), 2, "too large"),
        (win(b=1 << 16, hq=1 << 16), 2, "too large"), (win(ws=ctypes.c_void_p(8), nws=64), 1, "workspace"), (win(ws=p, nws=-1), 1, "workspace"),
        (pre(g=0), 1, "multiple"), (pre(g=3), 1, "multiple"), (pre(pl=-1), 1, "negative"), (pre(pk=None), 1, "null"), (pre(pl=1 << 31), 2, "too large"),
        (pre(plen=p, pdt=_lib.BOOL), 1, "prefix lengths"), (pre(pl=(1 << 30) - 1, c=(1 << 30) - 1), 2, "too large"),
    ]:
        assert rc == code, (rc, code, text)
    assert win(w=0) == 1 and "window" in _err()
    assert pre(g=3) == 1 and "multiple" in _err()
    # nothing to do: no launch, so safe without a GPU
    assert win(b=0) == 0 and win(sq=0) == 0 and win(d=0) == 0 and pre(g=0, b=0) == 0 and pre(hq=0) == 0

    def rot(d=8, rows=9, cols=4, axes=3, sections=(1, 1, 2), tdt=_lib.F32, dtype=_lib.BF16, q=p, pos=p, pdt=_lib.I64, s=5, q_out=None):
        return lib.ntops_rope_axes_qk(
            dtype, 2, s, 4, 2, d, q, st, p, st, tdt, p, 4, p, 4, rows, cols, axes, pos, pdt, st, len(sections), _lib.i64_array(sections), 0, p if q_out is None else q_out, st, p, st, None)

    for rc, code in [
        (rot(d=7), 1), (rot(d=514, cols=257, sections=(257,)), 2), (rot(cols=5), 1), (rot(axes=0), 1), (rot(sections=(1, 1, 1)), 1), (rot(sections=(3, -1, 2)), 1),
        (rot(sections=(1, 1, 1 << 62)), 1), (rot(tdt=_lib.F16), 1), (rot(dtype=_lib.F64), 2), (rot(q=None), 1), (rot(pos=None), 1), (rot(pdt=_lib.U8), 1),
        (rot(rows=-1), 1), (rot(s=1 << 50), 2),
    ]:
        assert rc == code
    assert rot(s=0) == 0


def test_rotary_sizes_whose_product_passes_64_bits():
    lib, p, st = _lib.load(), ctypes.c_void_p(256), _lib.i64_array((8, 8, 8, 1))
    for b, s in ((1 << 40, 1 << 24), (1 << 24, 1 << 40), (1 << 32, 1 << 32), (1 << 40, 1 << 40), (1 << 20, (1 << 20) + 1)):
        rc = lib.ntops_rope_axes_qk(
            _lib.BF16, b, s, 4, 2, 8, p, st, p, st, _lib.F32, p, 4, p, 4, 9, 4, 3, p, _lib.I64, st, 3, _lib.i64_array((1, 1, 2)), 0, p, st, p, st, None)
        assert rc == 2 and "too large" in _err()


def test_workspaces_of_refused_calls_are_empty():
    lib = _lib.load()
    for b, hq, hkv, sq, c, d, w, s in ((0, 4, 2, 1, 9, 8, 5, 0), (2, 3, 2, 1, 9, 8, 5, 0), (2, 4, 2, 1, 9, 300, 5, 0), (2, 4, 2, 1, 9, 8, 0, 0), (1 << 40, 4, 2, 1, 9, 8, 5, 0), (2, 4, 0, 1, 9, 8, 5, 0)):
        assert lib.ntops_sliding_window_attention_workspace(_lib.BF16, b, hq, hkv, sq, c, d, w, s) == 0
    assert lib.ntops_shared_prefix_attention_workspace(_lib.BF16, 3, 4, 4, 2, 1, 900, 9, 64) == 0
    assert lib.ntops_shared_prefix_attention_workspace(_lib.BF16, 0, 4, 4, 2, 1, 900, 9, 64) == 0
    # sizes that no machine holds: still no overflow
    for w in (1, 1 << 62):
        assert 0 <= lib.ntops_sliding_window_attention_workspace(_lib.BF16, 1, 8, 8, 1, 1 << 30, 128, w, 1 << 62) < 1 << 40


def test_oracle_identities():
    """A window past every key, and a prefix cut from a sequence, are causal attention;
    positions that agree on all axes rotate as one axis does."""
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(2, 4, 5, 8)), rng.normal(size=(2, 2, 9, 8)), rng.normal(size=(2, 2, 9, 8))
    whole = S.sliding_window_attention(q, k, v, 99, scale=0.5)[0]
    assert np.allclose(whole, S.sliding_window_attention(q, k, v, 1, 9, scale=0.5)[0])
    for i in range(2):
        cut = S.shared_prefix_attention(q[i : i + 1], k[i : i + 1, :, :3], v[i : i + 1, :, :3], k[i : i + 1, :, 3:], v[i : i + 1, :, 3:], scale=0.5)[0]
        assert np.allclose(whole[i], cut[0])
    own = S.sliding_window_attention(q, k, v, 1, scale=0.5)[0]
    assert np.allclose(own, np.repeat(v[:, :, 4:], 2, 1))  # each token sees itself alone
    # what is not seen does not count
    far = v.copy()
    far[:, :, :3] = np.nan
    assert np.allclose(S.sliding_window_attention(q, k, far, 2, scale=0.5)[0], S.sliding_window_attention(q, k, v, 2, scale=0.5)[0])
    x = rng.normal(size=(2, 5, 3, 8))
    angles = np.arange(20)[:, None] * 0.7 ** np.arange(4)
    row = rng.integers(0, 20, (2, 5))
    one = S.multi_axis_rotary_position_embedding(x, np.sin(angles), np.cos(angles), row[None], (4,), True)
    three = S.multi_axis_rotary_position_embedding(x, np.sin(angles), np.cos(angles), np.stack([row] * 3), (1, 0, 2, 1), True)
    assert np.allclose(one, three) and np.allclose((one**2).sum(-1), (x**2).sum(-1))
    bad = S.multi_axis_rotary_position_embedding(x, np.sin(angles), np.cos(angles), np.stack([row, row + 99]), (3, 1), False)
    assert np.isnan(bad).sum() == 2 * 5 * 3 * 2 and np.isnan(bad[..., [3, 7]]).all()


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (4, 2), (99, 0), (2, 99)])
def test_oracle_against_torch(window, sinks):
    """Both operators against torch's attention in 64 bits under a mask written key by key."""
    rng = np.random.default_rng(window)
    b, hq, h, sq, c, p, d = 3, 4, 2, 4, 9, 6, 8
    q, k, v = rng.normal(size=(b, hq, sq, d)), rng.normal(size=(b, h, c, d)), rng.normal(size=(b, h, c, d))
    pk, pv = rng.normal(size=(1, h, p, d)), rng.normal(size=(1, h, p, d))
    lengths, plen = [9, 2, 5], [4]

    def torch_attention(keys, vals, mask):
        keys, vals = (torch.from_numpy(np.repeat(t, hq // h, 1)) for t in (keys, vals))
        out = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q), keys, vals, torch.from_numpy(mask[:, None]), scale=0.7)
        return np.where(mask.any(-1)[:, None, :, None], out.numpy(), 0)

    mask = np.zeros((b, sq, c), bool)
    both = np.zeros((b, sq, p + c), bool)
    for i in range(b):
        for t in range(sq):
            at = lengths[i] - sq + t
            for j in range(c):
                mask[i, t, j] = j <= at and (j > at - window or j < sinks)
                both[i, t, p + j] = j <= at
            both[i, t, : plen[0]] = True
    got = S.sliding_window_attention(q, k, v, window, sinks, lengths, 0.7)[0]
    assert np.allclose(got, torch_attention(k, v, mask), atol=1e-12)
    got = S.shared_prefix_attention(q, pk, pv, k, v, plen, lengths, 0.7)[0]
    want = torch_attention(np.concatenate([np.repeat(pk, b, 0), k], 2), np.concatenate([np.repeat(pv, b, 0), v], 2), both)
    assert np.allclose(got, want, atol=1e-12)
