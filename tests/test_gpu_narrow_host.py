"""The native host path of the narrow-format operators against their Python
path: the same results bit for bit, the same refusals, and None (the Python
path) for what it does not take."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib

E4M3 = torch.float8_e4m3fn


def test_native_path_leaves_other_tensors_to_python():
    if _lib.fast is None:
        pytest.skip("the extension is not built")
    _lib.load()
    x = torch.randn(4, 64)
    u = torch.zeros(4, 32, dtype=torch.uint8)
    s = torch.zeros(4, 2, dtype=torch.uint8)

    class Sub(torch.Tensor):
        pass

    for t in (x, x.as_subclass(Sub), u, 3, None):
        assert _lib.fast.quantize_mxfp4(t) is None
        assert _lib.fast.dequantize_mxfp4(t, s, None, torch.bfloat16) is None
        assert _lib.fast.dequantize_mxfp4(u, t, None, torch.bfloat16) is None
        assert _lib.fast.mxfp4_mm(t, None, u, s, None, torch.bfloat16) is None
        assert _lib.fast.mxfp4_mm(u, s, u, t, None, torch.float16) is None
        assert _lib.fast.store_kv_cache(t, t, t, t, t, t, 0, None, 64) is None
        assert _lib.fast.kv_cache_attention(t, t, t, t, t, None, False, None, 64) is None
    assert _lib.fast.dequantize_mxfp4(u, s, None, "bf16") is None


def calls():
    torch.manual_seed(5)
    x = torch.randn(6, 200).bfloat16().cuda()
    codes, scales = nt.quantize_mxfp4(x)
    w, ws = nt.quantize_mxfp4(torch.randn(70, 200).cuda())
    b = torch.randn(70).bfloat16().cuda()
    for t in (x, x.float(), x.half(), x.view(2, 3, 200), x[:, :64], x[:, 1:], x[:0], x.t(), x.double()):
        yield lambda t=t: nt.quantize_mxfp4(t)
    for size in (None, 200, 193, 192, 224, 225, 0):
        for dtype in (torch.bfloat16, torch.float32, torch.float64):
            yield lambda size=size, dtype=dtype: nt.dequantize_mxfp4(codes, scales, size, dtype=dtype)
    yield lambda: nt.dequantize_mxfp4(codes[:, :96], scales[:, :6])
    yield lambda: nt.dequantize_mxfp4(codes, scales[:, :6])
    for a, sa in ((codes, scales), (x, None), (x.float(), None), (x[:, :100], None), (codes[:3], scales[:3]), (codes, None), (codes[:, :96], scales[:, :6]), (x.t(), None)):
        for bias in (None, b, b.float(), b[:5], torch.stack((b, b), 1)[:, 0]):
            yield lambda a=a, sa=sa, bias=bias: nt.mxfp4_mm(a, sa, w, ws, bias)
        yield lambda a=a, sa=sa: nt.mxfp4_mm(a, sa, w, ws, b.float(), dtype=torch.float32)
    yield lambda: nt.mxfp4_mm(codes[:0], scales[:0], w, ws)
    key = torch.randn(3, 2, 9, 64).bfloat16().cuda()
    kc, vc = (torch.zeros(3, 2, 50, 64, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.ones(3, 2, 4, device="cuda") for _ in range(2))
    pos = torch.tensor([0, 3, 30], device="cuda")
    for p in (0, 7, pos, pos.int(), pos.float(), pos[:2], None):
        for n in (None, pos, pos.int(), pos[::2]):
            for k in (key, key.transpose(1, 2).contiguous().transpose(1, 2), key[..., ::2], key.double()):

                def go(p=p, n=n, k=k):
                    nt.store_kv_cache(k, k, kc, vc, ks, vs, p, n, block_size=16)
                    out = [t.clone() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
                    nt.store_kv_cache(key.flip(2), key.flip(2), kc, vc, ks, vs, 0, block_size=16)
                    return out

                yield go
    for block in (16, 32, 24):
        yield lambda block=block: nt.kv_cache_attention(key, kc, vc, ks, vs, block_size=block)
    for q in (key, key.float(), key.repeat_interleave(2, 1), key[:, :, :1], key[:, :1], key[..., ::2], key[:2], key.transpose(1, 2).contiguous().transpose(1, 2), key[:, :, :0]):
        for n in (None, pos, pos.int(), pos.float()):
            for causal in (False, True, 1):
                for scale in (None, 0.5, 1, "no"):
                    yield lambda q=q, n=n, causal=causal, scale=scale: nt.kv_cache_attention(
                        q, kc, vc, ks, vs, n, causal, scale, block_size=16)


@pytest.mark.gpu
def test_native_and_python_paths_agree(monkeypatch):
    if _lib.fast is None:
        pytest.skip("the extension is not built")
    _lib.load()
    served = 0
    names = ("quantize_mxfp4", "dequantize_mxfp4", "mxfp4_mm", "store_kv_cache", "kv_cache_attention")

    class Counting:
        def __getattr__(self, name):
            fn = getattr(fast, name)

            def call(*a):
                nonlocal served
                r = fn(*a)
                served += name in names and r is not None
                return r

            return call

    fast = _lib.fast

    def run(call, path):
        monkeypatch.setattr(_lib, "fast", path)
        try:
            r = call()
        except Exception as e:
            return type(e), str(e)
        return [t.clone() for t in (r if isinstance(r, (tuple, list)) else (r,))]

    n = 0
    for call in calls():
        monkeypatch.setattr(_lib, "fast", fast)
        one, two = run(call, Counting()), run(call, None)
        n += 1
        assert type(one) is type(two), (one, two)
        if isinstance(one, tuple):
            assert one == two
            continue
        for x, y in zip(one, two):
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)
    assert n > 200 and served > 100


@pytest.mark.gpu
def test_device_and_streams_of_the_native_path():
    x = torch.randn(8, 512, device="cuda").bfloat16()
    w, ws = nt.quantize_mxfp4(torch.randn(96, 512, device="cuda"))
    want = nt.mxfp4_mm(x, None, w, ws)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([nt.mxfp4_mm(x, None, w, ws) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for many in outs for o in many)
