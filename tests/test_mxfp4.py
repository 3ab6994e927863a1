"""MXFP4 without a GPU: the oracle against closed forms, and what the entry
points refuse."""

import ctypes
import inspect

import numpy as np
import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib
from oracle import narrow as N


def test_oracle_rounds_to_the_nearest_code():
    grid = np.concatenate([N.E2M1, -N.E2M1])
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 96)) * np.exp(3 * rng.standard_normal((50, 1)))
    codes, scales = N.quantize_mxfp4(x)
    v = N.dequantize_mxfp4(codes, scales)
    s = np.repeat(np.exp2(scales.astype(float) - 127), 32, -1)
    best = np.abs(x[..., None] / s[..., None] - grid).min(-1)
    assert np.allclose(np.abs(x - v) / s, best, rtol=0, atol=1e-12)
    top = np.abs(x).reshape(50, 3, 32).max(-1)
    assert ((top / np.exp2(scales.astype(float) - 127) >= 4) & (top / np.exp2(scales.astype(float) - 127) < 8)).all()


def test_oracle_ties_go_to_the_even_code():
    x = np.zeros((1, 32))
    x[0, :9] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25]
    codes, scales = N.quantize_mxfp4(x)
    assert scales[0, 0] == 127
    assert N.dequantize_mxfp4(codes, scales)[0, :9].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0]


def test_oracle_packs_the_first_value_low():
    x = np.zeros((1, 32))
    x[0, :4] = [4.0, -0.5, 1.0, 6.0]
    codes, _ = N.quantize_mxfp4(x)
    assert codes[0, 0] == 6 | 9 << 4 and codes[0, 1] == 2 | 7 << 4


def test_oracle_zeros_and_not_finite():
    x = np.zeros((1, 96))
    x[0, 40], x[0, 70] = np.inf, np.nan
    codes, scales = N.quantize_mxfp4(x)
    assert scales.tolist() == [[0, 255, 255]] and not codes.any()


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
        ("_floor_log2(top) - 2, -127)", "_floor_log2(top) - 1, -127)"),
        ("(i % 2 == 1)", "(i % 2 == 0)"),
        ("code[..., 0] + 16 * code[..., 1]", "code[..., 1] + 16 * code[..., 0]"),
        ("np.where(bad, 255, e + 127)", "np.where(bad, 254, e + 127)"),
        ("np.where(nibbles < 8, 1.0, -1.0)", "np.where(nibbles > 8, 1.0, -1.0)"),
        ("[codes & 15, codes >> 4]", "[codes >> 4, codes & 15]"),
        ("E2M1[i] + E2M1[i + 1]) / 2", "E2M1[i] + 2 * E2M1[i + 1]) / 3"),
    ],
)
def test_oracle_checks_catch(right, wrong, monkeypatch):
    planted(monkeypatch, right, wrong)
    checks = (test_oracle_rounds_to_the_nearest_code, test_oracle_ties_go_to_the_even_code, test_oracle_packs_the_first_value_low, test_oracle_zeros_and_not_finite)
    assert any(catches(c) for c in checks)


def test_refusals():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="at least one dim"):
        nt.quantize_mxfp4(torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        nt.quantize_mxfp4(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="expected a GPU tensor"):
        nt.quantize_mxfp4(torch.zeros(2, 32))
    with pytest.raises(RuntimeError, match="codes"):
        nt.dequantize_mxfp4(u8(2, 32), u8(2, 1))
    with pytest.raises(RuntimeError, match="uint8"):
        nt.dequantize_mxfp4(u8(2, 32).int(), u8(2, 2))
    with pytest.raises(RuntimeError, match="blocks of 32"):
        nt.dequantize_mxfp4(u8(2, 32), u8(2, 2), 32)
    with pytest.raises(RuntimeError, match="blocks of 32"):
        nt.dequantize_mxfp4(u8(2, 32), u8(2, 2), 65)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        nt.dequantize_mxfp4(u8(2, 32), u8(2, 2), dtype=torch.float64)
    with pytest.raises(RuntimeError, match="2-D"):
        nt.mxfp4_mm(u8(1, 2, 32), u8(1, 2, 2), u8(4, 32), u8(4, 2))
    with pytest.raises(RuntimeError, match="expected a GPU tensor"):
        nt.mxfp4_mm(u8(2, 32), u8(2, 2), u8(4, 32), u8(4, 2))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        nt.mxfp4_mm(u8(2, 32), u8(2, 2), u8(4, 32), u8(4, 2), dtype=torch.float64)


P = ctypes.c_void_p


def _mm(lib, m=2, n=4, k=64, a=256, lda=32, as_=512, ldas=2, b=1024, ldb=32, bs=2048, ldbs=2, bias=None, out=4096, ldd=4, ws=None, wsb=0, dtype=_lib.BF16):
    return lib.ntops_mxfp4_mm(dtype, m, n, k, P(a), lda, P(as_), ldas, P(b), ldb, P(bs), ldbs, P(bias), P(out), ldd, P(ws), wsb, None)


def test_c_entry_points_refuse():
    lib = _lib.load()
    err = lambda: lib.ntops_last_error().decode()
    assert lib.ntops_quantize_mxfp4(_lib.BF16, -1, 32, P(256), 32, P(256), P(256), None) == 1 and "negative" in err()
    assert lib.ntops_quantize_mxfp4(_lib.F64, 1, 32, P(256), 32, P(256), P(256), None) == 2
    assert lib.ntops_quantize_mxfp4(_lib.BF16, 1, 32, None, 32, P(256), P(256), None) == 1 and "null" in err()
    assert lib.ntops_quantize_mxfp4(_lib.BF16, 1, 32, P(256), 32, P(258), P(256), None) == 1 and "aligned" in err()
    assert lib.ntops_quantize_mxfp4(_lib.BF16, 1 << 40, 1 << 40, P(256), 32, P(256), P(256), None) == 2
    assert lib.ntops_dequantize_mxfp4(_lib.BF16, 1, 32, P(256), 18, P(256), 1, P(256), None) == 1 and "aligned" in err()
    assert lib.ntops_dequantize_mxfp4(_lib.I32, 1, 32, P(256), 16, P(256), 1, P(256), None) == 2
    assert _mm(lib, m=-1) == 1
    assert _mm(lib, dtype=_lib.F64) == 2
    assert _mm(lib, a=264) == 1 and "16 bytes" in err()
    assert _mm(lib, ldb=40) == 1
    assert _mm(lib, ldas=-4) == 1 and "negative" in err()
    assert _mm(lib, out=None) == 1 and "null" in err()
    assert _mm(lib, k=1 << 40, lda=1 << 35, ldb=1 << 35) == 2 and "too large" in err()
    assert _mm(lib, ws=264) == 1 and "workspace" in err()
    assert _mm(lib, m=0) == 0 and lib.ntops_quantize_mxfp4(_lib.BF16, 0, 32, None, 32, None, None, None) == 0


def _linear(lib, x_dtype=_lib.BF16, dtype=_lib.BF16, m=2, n=4, k=64, x=256, ldx=64, b=1024, ldb=32, bs=2048, ldbs=2, bias=None, out=4096, ldd=4, ws=None, wsb=0):
    return lib.ntops_mxfp4_linear(x_dtype, dtype, m, n, k, P(x), ldx, P(b), ldb, P(bs), ldbs, P(bias), P(out), ldd, P(ws), wsb, None)


def test_linear_refuses():
    lib = _lib.load()
    err = lambda: lib.ntops_last_error().decode()
    for m in (2, 9):  # rounded by the product's kernel, and into the workspace
        assert _linear(lib, m=-m) == 1 and "negative" in err()
        assert _linear(lib, x_dtype=_lib.F64, m=m) == 2 and "input dtype" in err()
        ws = dict(ws=8192, wsb=1 << 20)
        assert _linear(lib, dtype=_lib.F64, m=m, **ws) == 2
        assert _linear(lib, x=None, m=m, **ws) == 1 and "null" in err()
        assert _linear(lib, out=None, m=m, **ws) == 1 and "null" in err()
        assert _linear(lib, b=None, m=m, **ws) == 1 and "null" in err()
        assert _linear(lib, b=1032, m=m, **ws) == 1 and "16 bytes" in err()
        assert _linear(lib, ldbs=-2, m=m, **ws) == 1 and "negative" in err()
        assert _linear(lib, m=m, k=1 << 40, ldx=1 << 40, **ws) == 2 and "too large" in err()
        assert _linear(lib, m=m, n=1 << 40, **ws) == 2 and "too large" in err()
        assert _linear(lib, m=0, x=None) == 0 and _linear(lib, n=0, m=m) == 0
    assert _linear(lib, m=9) == 1 and "workspace" in err()
    assert _linear(lib, m=9, ws=8192, wsb=9 * 34) == 1 and "workspace" in err()
    assert _linear(lib, m=9, ws=8196, wsb=1 << 20) == 1 and "workspace" in err()
    need = lib.ntops_mxfp4_linear_workspace
    assert need(_lib.BF16, 4, 4, 64, P(256), 64) == 0
    for args in ((_lib.F32, 4, 4, 64, P(256), 64), (_lib.BF16, 5, 4, 64, P(256), 64), (_lib.F16, 4, 4, 64, P(264), 64), (_lib.F16, 4, 4, 62, P(256), 64)):
        assert need(*args) >= args[1] * 34, args
    assert need(_lib.F16, 2, 4, 64, P(256), 65) >= 2 * 34 and need(_lib.F16, 1, 4, 64, P(256), 65) == 0
    assert need(_lib.BF16, 0, 4, 64, None, 64) == 0 and need(_lib.BF16, 4, 4, 0, None, 0) == 0
