"""The native host path of the windowed and shared-prefix attention and the multi-axis
rotary positions against their Python path: the same results bit for bit, the same
refusals, and None (the Python path) for what it does not take."""

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib


def test_native_path_leaves_other_tensors_to_python():
    if _lib.fast is None:
        pytest.skip("the extension is not built")
    _lib.load()
    x = torch.randn(2, 2, 4, 64)

    class Sub(torch.Tensor):
        pass

    for t in (x, x.as_subclass(Sub), 3, None):
        assert _lib.fast.sliding_window_attention(t, t, t, 5, 0, None, None) is None
        assert _lib.fast.shared_prefix_attention(t, t, t, t, t, None, None, None) is None
        assert _lib.fast.rope_axes_qk(t, t, t, t, t, (32,), True) is None
    assert _lib.fast.sliding_window_attention(x, x, x, 1 << 70, 0, None, None) is None


def calls():
    torch.manual_seed(7)
    key = torch.randn(4, 2, 50, 64).bfloat16().cuda()
    value = torch.randn(4, 2, 50, 64).bfloat16().cuda()
    pk, pv = torch.randn(2, 2, 70, 64).bfloat16().cuda(), torch.randn(2, 2, 70, 64).bfloat16().cuda()
    n = torch.tensor([50, 3, 20, 0], device="cuda")
    queries = [key[:, :, :5], key.repeat_interleave(3, 1)[:, :, :40], key[:, :, :5].float(), key[:, :1, :3], key[..., ::2], key[:2], key[:, :, :0],
               key[:, :, :5].transpose(1, 2).contiguous().transpose(1, 2), key[:, :, :5].double(), key[0]]
    for q in queries:
        for lengths in (None, n, n.int(), n.float(), n[::2], torch.stack((n, n), 1)[:, 0]):
            for window, sinks in ((7, 2), (1, 0), (0, 1), (5, -1), (1 << 70, 1 << 70), (2.5, 0), (True, 0), (7, None)):
                yield lambda q=q, lengths=lengths, window=window, sinks=sinks: nt.sliding_window_attention(q, key, value, window, sinks, lengths)
            for scale in (None, 0.5, 1, "no"):
                yield lambda q=q, lengths=lengths, scale=scale: nt.shared_prefix_attention(q, pk, pv, key, value, n[:2], lengths, scale)
                yield lambda q=q, lengths=lengths, scale=scale: nt.sliding_window_attention(q, key, value, 9, 3, lengths, scale)
        for k, v in ((key[:, :, :0], value[:, :, :0]), (key.float(), value), (key[..., ::2], value[..., ::2]), (key[:, :1], value[:, :1]), (key, value[:, :, :9]), (key.cpu(), value)):
            yield lambda q=q, k=k, v=v: nt.sliding_window_attention(q, k, v, 9, 3)
            yield lambda q=q, k=k, v=v: nt.shared_prefix_attention(q, k[:2], v[:2], key, value)
            yield lambda q=q, k=k, v=v: nt.shared_prefix_attention(q, pk, pv, k, v)
            yield lambda q=q, k=k, v=v: nt.shared_prefix_attention(q, k[:3], v[:3], key, value, n[:3])
    q, k = torch.randn(2, 9, 4, 64).bfloat16().cuda(), torch.randn(2, 9, 2, 64).bfloat16().cuda()
    sin, cos = torch.randn(30, 32).cuda(), torch.randn(30, 32).cuda()
    pos = torch.randint(0, 30, (3, 2, 9)).cuda()
    for x in (q, q.transpose(1, 2), q.float(), q.double(), q[:, :3], q[..., :63], q[:, :, :, ::2], q.transpose(1, 2).contiguous().transpose(1, 2), q[0]):
        for p in (pos, pos.int(), pos[:, :1].expand(3, 2, 9), pos.float(), pos[:, :1], pos[0]):
            for sections in ((8, 12, 12), [8, 12, 12], (32,), (1,) * 32, (8, 12), (33, -1, 0), (8.0, 12, 12), 32, range(0)):
                yield lambda x=x, p=p, sections=sections: nt.multi_axis_rotary_position_embedding_qk(x, k, sin, cos, p, sections, False)
    for s, c in ((sin.bfloat16(), cos.bfloat16()), (sin.double(), cos.double()), (sin.bfloat16(), cos), (sin[:, ::2], cos[:, ::2]), (sin, cos[:9]), (sin.t().contiguous().t(), cos), (torch.cat((sin, cos), 1),) * 2, (sin[:0], cos[:0])):
        for interleaved in (True, False, 1):
            yield lambda s=s, c=c, interleaved=interleaved: nt.multi_axis_rotary_position_embedding_qk(q, k, s, c, pos, (8, 12, 12), interleaved)


@pytest.mark.gpu
def test_native_and_python_paths_agree(monkeypatch):
    if _lib.fast is None:
        pytest.skip("the extension is not built")
    _lib.load()
    served = 0
    fast = _lib.fast

    class Counting:
        def __getattr__(self, name):
            def call(*a):
                nonlocal served
                r = getattr(fast, name)(*a)
                served += r is not None
                return r

            return call

    def run(call, path):
        monkeypatch.setattr(_lib, "fast", path)
        try:
            r = call()
        except Exception as e:
            return type(e), str(e)
        return [t.clone() for t in (r if isinstance(r, (tuple, list)) else (r,))]

    n = 0
    for call in calls():
        one, two = run(call, Counting()), run(call, None)
        n += 1
        assert type(one) is type(two), (one, two)
        if isinstance(one, tuple):
            assert one == two
            continue
        for x, y in zip(one, two):
            assert x.dtype == y.dtype and x.shape == y.shape
            assert torch.equal(torch.nan_to_num(x, nan=-99.0), torch.nan_to_num(y, nan=-99.0))
    assert n > 1000 and served > 100, (n, served)


@pytest.mark.gpu
def test_gradients_are_not_recorded_and_inputs_stay():
    q = torch.randn(2, 4, 3, 64, device="cuda", requires_grad=True)
    k, v = torch.randn(2, 2, 30, 64, device="cuda", requires_grad=True), torch.randn(2, 2, 30, 64, device="cuda")
    before = [t.detach().clone() for t in (q, k, v)]
    for out in (nt.sliding_window_attention(q, k, v, 9), nt.shared_prefix_attention(q, k[:1], v[:1], k, v)):
        assert not out.requires_grad and torch.isfinite(out).all()
    assert all(torch.equal(x, y) for x, y in zip(before, (q, k, v)))
