"""The key / value cache in 8 bits without a GPU: the oracle against torch's own
e4m3 and attention, and what the entry points refuse."""

import ctypes
import inspect

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import narrow as N

E4M3 = torch.float8_e4m3fn


def test_oracle_rounds_as_torch_does():
    x = torch.cat([torch.randn(20000) * torch.exp(3 * torch.randn(20000)), torch.arange(-4000, 4000) / 2**11, torch.tensor([448.0, 464.0, -0.0, float("nan"), float("inf")])])
    x = x[~(x.abs() > 464) | ~torch.isfinite(x)]
    assert np.array_equal(np.nan_to_num(N.e4m3(x.numpy()), nan=-1.0), np.nan_to_num(x.to(E4M3).double().numpy(), nan=-1.0))


def test_oracle_scale_is_the_least():
    top = np.concatenate([np.exp(np.random.default_rng(0).standard_normal(1000) * 10), [448.0, 449.0, 448 * 2.0**-40, 224.0, 1e-45, 0.0]])
    s = N.cache_scale(top)
    assert (top <= 448 * s).all() and ((top > 224 * s) | (s == 2.0**-126)).all()


def test_oracle_store_reads_back():
    rng = np.random.default_rng(1)
    cache, scale = np.zeros((1, 2, 50, 8)), np.zeros((1, 2, 4))
    seen = []
    for t in range(50):
        x = rng.standard_normal((1, 2, 1, 8)) * 2.0 ** rng.integers(-3, 4)
        seen.append(x)
        cache, scale = N.store_kv_cache(x, cache, scale, [t], [1], 16)
    x = np.concatenate(seen, 2)
    back = cache * scale[..., np.arange(50) // 16][..., None]
    top = np.abs(x).max((2, 3), keepdims=True)
    assert (np.abs(back - x) <= 2.0**-4 * np.abs(x) + 2.0**-10 * np.repeat(scale, 16, -1)[..., :50, None] * 3).all() and top.all()


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((2, 4, 3, 8)), rng.standard_normal((2, 2, 20, 8)), rng.standard_normal((2, 2, 20, 8))
    ks, vs = np.full((2, 2, 2), 0.5), np.full((2, 2, 2), 2.0)
    out = N.kv_cache_attention(q, k, v, ks, vs, [20, 2], 16, True, 0.3)
    kk, vv = (torch.from_numpy(x).repeat_interleave(2, 1) for x in (k * 0.5, v * 2))
    mask = torch.ones(3, 20, dtype=torch.bool).tril(17)
    want = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q), kk, vv, mask, scale=0.3)
    assert np.allclose(out[0], want[0].numpy())
    assert not out[1, :, 0].any() and np.allclose(out[1, :, 1], vv[1, :, 0].numpy())


def test_oracle_attention_scales_each_block():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((1, 2, 2, 8)), rng.standard_normal((1, 1, 40, 8)), rng.standard_normal((1, 1, 40, 8))
    ks, vs = np.array([[[0.5, 2.0, 0.125]]]), np.array([[[4.0, 0.25, 1.5]]])
    out = N.kv_cache_attention(q, k, v, ks, vs, [37], 16, False, 0.5)
    at = np.arange(37) // 16
    kk, vv = (torch.from_numpy(x[:, :, :37] * s[..., at][..., None]).expand(1, 2, 37, 8) for x, s in ((k, ks), (v, vs)))
    assert np.allclose(out, torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q), kk, vv, scale=0.5).numpy())


def planted(monkeypatch, right, wrong):
    """The oracle with one mistake in it."""
    source = inspect.getsource(N)
    assert source.count(right) == 1
    names = {}
    exec(compile(source.replace(right, wrong), "planted", "exec"), names)
    for name, value in names.items():
        if inspect.isfunction(value):
            monkeypatch.setattr(N, name, value)


def catches(check):
    try:
        check()
    except AssertionError:
        return True
    return False


@pytest.mark.parametrize(
    "right,wrong",
    [
        ("-6).astype(np.float64) - 3", "-5).astype(np.float64) - 3"),
        ("np.rint(a / unit)", "np.floor(a / unit)"),
        ("1.0)) - 8, -126)", "1.0)) - 7, -126)"),
        ("(old / s)", "(s / old)"),
        ("if old > s:", "if old < s:"),
        ("np.arange(Sq)[:, None] + n - Sq if", "np.arange(Sq)[:, None] + n - Sq - 1 if"),
        ("g = h // group", "g = h % k.shape[1]"),
        ("[at // block][:, None]\n            s = ", "[at // block - 1][:, None]\n            s = "),
    ],
)
def test_oracle_checks_catch(right, wrong, monkeypatch):
    planted(monkeypatch, right, wrong)
    checks = (test_oracle_rounds_as_torch_does, test_oracle_scale_is_the_least, test_oracle_store_reads_back, test_oracle_attention_is_softmax,
              test_oracle_attention_scales_each_block)
    assert any(catches(c) for c in checks)


def caches(b=2, h=2, c=40, d=16, block=16, dtype=E4M3):
    kc, vc = (torch.zeros(b, h, c, d, dtype=torch.uint8).view(dtype) for _ in range(2))
    return [kc, vc, torch.ones(b, h, -(-c // block)), torch.ones(b, h, -(-c // block))]


def refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def test_store_refusals():
    x = torch.zeros(2, 2, 3, 16)
    c = caches()
    go = lambda *a, block=16, **k: (lambda: nt.store_kv_cache(*a, block_size=block, **k))
    refuses("power of two", go(x, x, *c, 0, block=24))
    refuses("power of two", go(x, x, *c, 0, block=8))
    refuses("scales of shape", go(x, x, *c, 0, block=32))
    refuses("float8_e4m3fn", go(x, x, *caches(dtype=torch.uint8), 0))
    refuses("4-D caches", go(x, x, c[0], c[1][:, :, :30], *c[2:], 0))
    refuses("do not fit", go(x[..., :8], x[..., :8], *c, 0))
    refuses("do not fit", go(x, x[:, :, :2], *c, 0))
    refuses("do not fit", go(x[:1], x[:1], *c, 0))
    refuses("unsupported dtypes", go(x.double(), x.double(), *c, 0))
    refuses("unsupported dtypes", go(x, x.half(), *c, 0))
    refuses("positions", go(x, x, *c, torch.zeros(3, dtype=torch.int32)))
    refuses("positions", go(x, x, *c, torch.zeros(2)))
    refuses("lengths", go(x, x, *c, 0, torch.zeros(2, 1, dtype=torch.int64)))
    refuses("share memory", go(x, x, c[0][:1].expand(2, -1, -1, -1), *c[1:], 0))
    refuses("unit stride", go(x, x, c[0].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3).view(E4M3), *c[1:], 0))
    refuses("expected a GPU tensor", go(x, x, *c, 0))


def test_attention_refusals():
    q = torch.zeros(2, 4, 3, 16)
    c = caches()
    go = lambda *a, block=16, **k: (lambda: nt.kv_cache_attention(*a, block_size=block, **k))
    refuses("power of two", go(q, *c, block=0))
    refuses("does not fit", go(q[..., :8], *c))
    refuses("does not fit", go(q[0], *c))
    refuses("does not fit", go(q[:1], *c))
    refuses("multiple", go(q[:, :3], *c))
    refuses("unsupported dtype", go(q.double(), *c))
    refuses("lengths", go(q, *c, torch.zeros(2)))
    refuses("lengths", go(q, *c, torch.zeros(1, dtype=torch.int32)))
    refuses("expected a GPU tensor", go(q, *c))


P = ctypes.c_void_p


def test_c_entry_points_refuse():
    lib = _lib.load()
    err = lambda: lib.ntops_last_error().decode()
    s4, s3 = _lib.i64_array((640, 320, 16, 1)), _lib.i64_array((6, 3, 1))
    bad4 = _lib.i64_array((640, 320, 1, 40))

    def store(dtype=_lib.BF16, b=2, h=2, s=3, d=16, c=40, block=16, key=256, ks=s4, cs=s4, pos=None, pdt=0, ldt=0, lens=None):
        return lib.ntops_store_kv_cache(dtype, b, h, s, d, c, block, P(key), ks, P(512), s4, P(1024), cs, P(2048), s4, P(4096), s3, P(8192), s3, P(pos), pdt, 0, P(lens), ldt, None)

    assert store(b=-1) == 1 and "negative" in err()
    assert store(block=48) == 1 and "power of two" in err()
    assert store(dtype=_lib.F64) == 2
    assert store(key=None) == 1 and "null" in err()
    assert store(ks=bad4) == 1 and "unit strides" in err()
    assert store(cs=bad4) == 1 and "unit strides" in err()
    assert store(pos=256, pdt=_lib.F32) == 1 and "I32 or I64" in err()
    assert store(lens=256, ldt=_lib.I16) == 1
    assert store(d=1 << 20) == 2 and store(b=1 << 33) == 2 and store(h=70000) == 2
    assert store(b=0, key=None) == 0 and store(s=0, key=None) == 0

    def attend(dtype=_lib.BF16, b=2, hq=4, h=2, sq=3, c=40, d=16, block=16, q=256, qs=s4, cs=s4, lens=None, ldt=0, causal=0, out=512):
        return lib.ntops_kv_cache_attention(dtype, b, hq, h, sq, c, d, block, P(q), qs, P(1024), cs, P(2048), s4, P(4096), s3, P(8192), s3, P(lens), ldt, causal, 0.5, P(out), s4, None, 0, None)

    assert attend(sq=-1) == 1
    assert attend(dtype=_lib.F64) == 2
    assert attend(block=17) == 1 and "power of two" in err()
    assert attend(hq=3) == 1 and "multiple" in err()
    assert attend(h=0) == 1
    assert attend(q=None) == 1 and "null" in err()
    assert attend(out=None) == 1
    assert attend(qs=bad4) == 1 and "unit strides" in err()
    assert attend(cs=bad4) == 1 and "unit strides" in err()
    assert attend(lens=256, ldt=_lib.F16) == 1 and "I32 or I64" in err()
    assert attend(causal=2) == 1
    assert attend(d=257) == 2 and "head dim" in err()
    assert attend(b=0, q=None) == 0 and attend(sq=0, q=None) == 0


def test_store_refuses_one_cache_for_both():
    lib = _lib.load()
    arr = lambda *v: (ctypes.c_int64 * len(v))(*v)
    s4, s3 = arr(2048, 1024, 16, 1), arr(8, 4, 1)

    def go(vc=2048, vs=8192):
        return lib.ntops_store_kv_cache(_lib.BF16, 2, 2, 1, 16, 64, 16, P(256), s4, P(512), s4, P(1024), s4, P(vc), s4, P(4096), s3, P(vs), s3, None, 0, 0, None, 0, None)

    for same in (dict(vc=1024), dict(vs=4096)):
        assert go(**same) == 1 and "share" in lib.ntops_last_error().decode()
