"""sliding_window_attention -- attention in which a token sees the last `window`
tokens, itself among them, and the first `sinks` tokens of its sequence.

No ntops counterpart (torch/scaled_dot_product_attention.py:10-108 takes a window
as an explicit mask and reads every key).  query (batch, query heads, tokens,
head_dim); key and value (batch, heads, capacity, head_dim) of the same type, of
which sequence b holds its first lengths[b] tokens (int32 or int64 (batch,); None:
all; read on the device and cut to the capacity).  The last query row is the
sequence's last token: row i is its token p = lengths[b] - tokens + i, and sees the
keys j <= p with j > p - window or j < sinks.  Query head h reads head h // (query
heads / heads).  A row that sees no key is 0; what a row does not see does not reach
it, NaNs and infinities included.  Prompts that are padded in front have rows before
their first token, which are 0; for prompts padded at their end, lengths of `tokens`
leave token i at row i.  scale defaults to 1 / sqrt(head_dim).

float16, bfloat16 or float32, head dims up to 256; multiples of 8 (float32: of 4) run
on the matrix cores."""

import math
import operator

import torch

from ntops_amd import _lib
from ntops_amd.torch.store_kv_cache import _check_index
from ntops_amd.torch.utils import _DeviceGuard, _contiguous, _strides


def _check_attention(query, key, value, what):
    """The shape (batch, query heads, heads, tokens, capacity, head_dim)."""
    if query.dim() != 4 or key.dim() != 4 or key.shape != value.shape:
        raise RuntimeError(
            f"{what}: expected a 4-D query and key and value of one 4-D shape, got {tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}")
    if query.dtype not in (torch.float32, torch.float16, torch.bfloat16) or key.dtype != query.dtype or value.dtype != query.dtype:
        raise RuntimeError(f"{what}: expected one of float32, float16 and bfloat16, got {query.dtype}, {key.dtype} and {value.dtype}")
    b, hq, sq, d = query.shape
    if key.shape[0] != b or key.shape[3] != d:
        raise RuntimeError(f"{what}: query {tuple(query.shape)} does not fit keys of shape {tuple(key.shape)}")
    hkv = key.shape[1]
    if hkv == 0 or hq % hkv:
        raise RuntimeError(f"{what}: {hq} query heads are not a multiple of {hkv} key / value heads")
    return b, hq, hkv, sq, key.shape[2], d


def _index_args(t):
    return (None, 0) if t is None else (t.data_ptr(), _lib.dtype_code(t.dtype))


def sliding_window_attention(query, key, value, window, sinks=0, lengths=None, scale=None):
    if _lib.fast is not None:
        r = _lib.fast.sliding_window_attention(query, key, value, window, sinks, lengths, scale)
        if r is not None:
            return r
    what = "sliding_window_attention"
    b, hq, hkv, sq, c, d = _check_attention(query, key, value, what)
    window, sinks = (min(operator.index(n), 1 << 62) for n in (window, sinks))
    if window < 1 or sinks < 0:
        raise RuntimeError(f"{what}: expected a window of at least 1 and sinks of at least 0, got {window} and {sinks}")
    if lengths is not None:
        _check_index(lengths, b, "lengths", what)
    dev = _lib.require_cuda(query, key, value, lengths)
    if scale is None:
        scale = 1 / math.sqrt(d) if d else 1.0
    output = torch.empty(query.shape, dtype=query.dtype, device=dev)
    lib = _lib.load()
    dt = _lib.dtype_code(query.dtype)
    with _DeviceGuard(dev):
        if query.stride(3) != 1 and d > 1:
            query = _contiguous(query)
        lengths = None if lengths is None else _contiguous(lengths)
        ws_bytes = lib.ntops_sliding_window_attention_workspace(dt, b, hq, hkv, sq, c, d, window, sinks)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        rc = lib.ntops_sliding_window_attention(
            dt, b, hq, hkv, sq, c, d, query.data_ptr(), _strides(query), key.data_ptr(), _strides(key),
            value.data_ptr(), _strides(value), *_index_args(lengths), window, sinks, float(scale),
            output.data_ptr(), _strides(output), None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream_of(output))
    _lib.check(rc, "ntops_amd.sliding_window_attention")
    return output
