"""shared_prefix_attention -- attention of a batch whose sequences share their first
tokens: a system prompt, a document, or the prompt of several samples.

No ntops counterpart (torch/scaled_dot_product_attention.py:10-108 would hold the
prefix's keys and values once per sequence, and read them as often).  prefix_key and
prefix_value (groups, heads, prefix capacity, head_dim) hold the prefixes, of
prefix_lengths[g] tokens each ((groups,) int32 or int64; None: all); sequence b of
the batch shares that of group b // (batch / groups).  key and value (batch, heads,
capacity, head_dim) hold what follows in each sequence, lengths[b] tokens of it
((batch,); None: all).  Lengths are read on the device and cut to the capacity.

query (batch, query heads, tokens, head_dim): the last row is the sequence's last
token.  Row i sees the whole prefix and its own sequence's tokens up to
lengths[b] - tokens + i -- none of them where that is negative.  Query head h reads
head h // (query heads / heads).  A row that sees no key is 0; what a row does not
see does not reach it, NaNs and infinities included.  scale defaults to
1 / sqrt(head_dim).

float16, bfloat16 or float32, head dims up to 256; multiples of 8 (float32: of 4) run
on the matrix cores."""

import math

import torch

from ntops_amd import _lib
from ntops_amd.torch.sliding_window_attention import _check_attention, _index_args
from ntops_amd.torch.store_kv_cache import _check_index
from ntops_amd.torch.utils import _DeviceGuard, _contiguous, _strides


def shared_prefix_attention(query, prefix_key, prefix_value, key, value, prefix_lengths=None, lengths=None, scale=None):
    if _lib.fast is not None:
        r = _lib.fast.shared_prefix_attention(query, prefix_key, prefix_value, key, value, prefix_lengths, lengths, scale)
        if r is not None:
            return r
    what = "shared_prefix_attention"
    b, hq, hkv, sq, c, d = _check_attention(query, key, value, what)
    if prefix_key.dim() != 4 or prefix_key.shape != prefix_value.shape or prefix_key.shape[1] != hkv or prefix_key.shape[3] != d:
        raise RuntimeError(
            f"{what}: prefixes of shapes {tuple(prefix_key.shape)} and {tuple(prefix_value.shape)} do not fit keys of shape {tuple(key.shape)}")
    if prefix_key.dtype != query.dtype or prefix_value.dtype != query.dtype:
        raise RuntimeError(f"{what}: expected prefixes of {query.dtype}, got {prefix_key.dtype} and {prefix_value.dtype}")
    groups, _, p, _ = prefix_key.shape
    if groups == 0 and b > 0 or groups and b % groups:
        raise RuntimeError(f"{what}: a batch of {b} is not a multiple of {groups} prefixes")
    if prefix_lengths is not None:
        _check_index(prefix_lengths, groups, "prefix_lengths", what)
    if lengths is not None:
        _check_index(lengths, b, "lengths", what)
    dev = _lib.require_cuda(query, prefix_key, prefix_value, key, value, prefix_lengths, lengths)
    if scale is None:
        scale = 1 / math.sqrt(d) if d else 1.0
    output = torch.empty(query.shape, dtype=query.dtype, device=dev)
    lib = _lib.load()
    dt = _lib.dtype_code(query.dtype)
    with _DeviceGuard(dev):
        if query.stride(3) != 1 and d > 1:
            query = _contiguous(query)
        prefix_lengths, lengths = (None if t is None else _contiguous(t) for t in (prefix_lengths, lengths))
        ws_bytes = lib.ntops_shared_prefix_attention_workspace(dt, groups, b, hq, hkv, sq, p, c, d)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        rc = lib.ntops_shared_prefix_attention(
            dt, groups, b, hq, hkv, sq, p, c, d, query.data_ptr(), _strides(query),
            prefix_key.data_ptr(), _strides(prefix_key), prefix_value.data_ptr(), _strides(prefix_value),
            *_index_args(prefix_lengths), key.data_ptr(), _strides(key), value.data_ptr(), _strides(value),
            *_index_args(lengths), float(scale), output.data_ptr(), _strides(output),
            None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream_of(output))
    _lib.check(rc, "ntops_amd.shared_prefix_attention")
    return output
