"""What multi_axis_rotary_position_embedding_qk refuses to rotate in place: elements that
the query and the key share, or that one of them holds twice.  By addresses counted one
by one; on tensors of the CPU, so a call that is not refused ends at "GPU tensor"."""

import ctypes
import random

import pytest
import torch

import ntops_amd.torch as nt
from ntops_amd import _lib


def verdict(q, k, inplace=True):
    """What the wrapper says of the pair: "itself", "twice" or None."""
    b, s, _, d = q.shape
    tables = torch.zeros(3, d // 2), torch.zeros(3, d // 2)
    with pytest.raises(RuntimeError) as e:
        nt.multi_axis_rotary_position_embedding_qk(q, k, *tables, torch.zeros(1, b, s, dtype=torch.int64), (d // 2,), inplace=inplace)
    text = str(e.value)
    assert "GPU tensor" in text or "share memory" in text or "twice" in text
    return "itself" if "share memory" in text else "twice" if "twice" in text else None


def refused(dtype, q, q_out, k, k_out):
    """Whether the C entry refuses these, given as (address, shape, strides), of which no
    memory is read; only for calls that it has to refuse."""
    st = _lib.i64_array
    (b, s, hq, d), hk = q[1], k[1][2]
    t = ctypes.c_void_p(64)
    rc = _lib.load().ntops_rope_axes_qk(
        dtype, b, s, hq, hk, d, q[0], st(q[2]), k[0], st(k[2]), _lib.F32, t, d // 2, t, d // 2, 3, d // 2, 1, t, _lib.I64, st((0, 0, 0)), 1, st((d // 2,)), 0,
        q_out[0], st(q_out[2]), k_out[0], st(k_out[2]), None)
    return rc == 1 and "share" in _lib.load().ntops_last_error().decode()


def c_form(x):
    return x.data_ptr(), tuple(x.shape), x.stride()


def pairs():
    x, z = torch.zeros(3, 6, 8, 64), torch.zeros(2, 5, 4, 128)
    yield x[:, :-1], x[:, 1:], "twice"  # tokens
    yield x[:2], x[1:], "twice"  # sequences
    yield z[..., :64], z[..., 32:96], "twice"  # columns
    yield x[:, :, 0:8:2], x[:, :, 2:5], "twice"  # every second head
    yield x[:, :, :4], x[:, :, 3:], "twice"
    yield x.transpose(1, 2)[:, :6, :6], x[:, :6, :6], "twice"
    yield x.flip(1)[:, :1].as_strided((3, 1, 8, 64), x.stride()), torch.zeros(3, 1, 2, 64), None
    yield x[:, :, :1].expand(3, 6, 4, 64), torch.zeros(3, 6, 2, 64), "itself"
    yield torch.zeros(9).as_strided((1, 2, 2, 4), (0, 2, 1, 1)), torch.zeros(1, 2, 1, 4), "itself"
    yield torch.zeros(1, 2, 1, 4), torch.zeros(99).as_strided((1, 2, 3, 4), (7, 9, 3, 1)), "itself"
    # apart: packed heads, one head's query, key and value side by side, heads in turn, halves
    yield x[:, :, :5], x[:, :, 5:7], None
    yield x[:, :, 6:], x[:, :, :6], None
    h = torch.zeros(2, 5, 8, 3, 64)
    yield h[:, :, :, 0], h[:, :, :, 1], None
    yield x[:, :, 0::2], x[:, :, 1::2], None
    yield x[:, :, 0:8:2], x[:, :, 3:4], None
    yield z[..., :64], z[..., 64:], None
    yield z[..., 0::2], z[..., 1::2], None
    yield x[:1], x[1:2], None
    yield x[:, :3], x[:, 3:], None
    yield x.permute(0, 2, 1, 3)[:, :, :2], x.permute(0, 2, 1, 3)[:, :, 2:], None
    yield x.permute(1, 2, 3, 0)[..., :2], x.permute(1, 2, 3, 0)[..., 1:], "twice"
    yield x, x.clone(), None
    yield x[:, :, :0], x, None
    one = torch.zeros(1, 1, 6, 64)  # strides of dims of one element do not count
    yield one[:, :, :4], one[:, :, 4:].as_strided((1, 1, 2, 64), (1, 3, 64, 1)), None


def test_pairs():
    seen = set()
    for q, k, want in pairs():
        assert verdict(q, k) == want, (q.shape, q.stride(), k.shape, k.stride())
        assert verdict(q, k, inplace=False) is None
        if want:
            assert refused(_lib.F32, c_form(q), c_form(q), c_form(k), c_form(k))
        seen.add(want)
    assert seen == {None, "itself", "twice"}


def addresses(place, shape, strides):
    out = [place]
    for n, s in zip(shape, strides):
        out = [a + i * s for a in out for i in range(n)]
    return out


def test_every_small_layout():
    """Random layouts in a few hundred elements against their addresses, one by one."""
    rng = random.Random(1)
    base = torch.zeros(4000)
    count = {"itself": 0, "twice": 0, None: 0}
    for _ in range(3000):
        b, s, d = rng.choice([1, 1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([2, 4])
        dims = []
        for heads in (rng.choice([1, 2, 3]), rng.choice([1, 2, 5])):
            shape = (b, s, heads, d)
            if dims and rng.random() < 0.5:
                strides = dims[0][2]
            elif rng.random() < 0.6:  # nested, in some order, with gaps
                strides, step = [0] * 4, rng.choice([1, 1, 2])
                for i in rng.sample(range(4), 4):
                    strides[i] = step
                    step *= shape[i] + rng.choice([0, 0, 1, heads])
            else:
                strides = [rng.randrange(0, 12) for _ in range(4)]
            dims.append((rng.randrange(60), shape, tuple(strides)))
        at = [addresses(*x) for x in dims]
        want = "itself" if any(len(set(a)) < len(a) for a in at) else "twice" if set(at[0]) & set(at[1]) else None
        q, k = (base.as_strided(shape, strides, place) for place, shape, strides in dims)
        assert verdict(q, k) == want, dims
        count[want] += 1
        if want:
            assert refused(_lib.F32, c_form(q), c_form(q), c_form(k), c_form(k)), dims
    assert min(count.values()) > 300, count


def test_c_entry_refuses_results_that_meet():
    """Of calls out of place: results that meet each other, the other tensor, or otherwise
    their own."""
    x = torch.zeros(2, 3, 8, 4, dtype=torch.bfloat16)
    y = torch.zeros(2, 3, 8, 4, dtype=torch.bfloat16)
    q, k, qo, ko = (c_form(t) for t in (x[:, :, :4], x[:, :, 4:], y[:, :, :4], y[:, :, 4:]))
    shift = c_form(y[:, :, 3:7])
    back = (qo[0] + 2 * 3 * 32, qo[1], (96, -32, 4, 1))  # a sequence's tokens from the last one on: of both sequences
    for args in (
        (q, shift, k, ko), (q, c_form(x[:, :, 3:7]), k, ko), (q, c_form(x[:, :, 1:5]), k, ko), (q, qo, k, c_form(x[:, :, :4])), (q, qo, k, qo),
        (q, (qo[0], qo[1], (96, 32, 0, 1)), k, ko), (q, (qo[0], qo[1], (96, 32, 4, 0)), k, ko), (q, (qo[0] + 1, *qo[1:]), k, qo), (q, back, k, qo),
    ):
        assert refused(_lib.BF16, *args), args


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pairs_on_the_gpu(dtype, path, monkeypatch):
    """What is refused there too, and what is not: rotated in place as out of place, each
    memory once, and nothing else written."""
    if path == "python":
        monkeypatch.setattr(_lib, "fast", None)
    for q, k, want in pairs():
        (b, s, _, d), whole = q.shape, {}
        for t in (q, k):  # one tensor of the GPU for each storage
            of = t.untyped_storage()
            whole.setdefault(of.data_ptr(), torch.randn(of.nbytes() // 4).to(dtype).cuda())
        q, k = (whole[t.untyped_storage().data_ptr()].as_strided(t.shape, t.stride(), t.storage_offset()) for t in (q, k))
        tables = torch.randn(30, d // 2, device="cuda"), torch.randn(30, d // 2, device="cuda")
        args = (*tables, torch.randint(0, 30, (1, b, s), device="cuda"), (d // 2,))
        if want:
            with pytest.raises(RuntimeError, match="share memory" if want == "itself" else "twice"):
                nt.multi_axis_rotary_position_embedding_qk(q, k, *args, inplace=True)
            continue
        after = nt.multi_axis_rotary_position_embedding_qk(q, k, *args)
        copies = {t.data_ptr(): t.clone() for t in whole.values()}
        for t, y in zip((q, k), after):
            copies[t.untyped_storage().data_ptr()].as_strided(t.shape, t.stride(), t.storage_offset()).copy_(y)
        got = nt.multi_axis_rotary_position_embedding_qk(q, k, *args, inplace=True)
        assert got[0] is q and got[1] is k
        assert all(torch.equal(t, copies[t.data_ptr()]) for t in whole.values())
