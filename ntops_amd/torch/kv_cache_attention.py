"""kv_cache_attention -- attention over a cache held in 8 bits (see
store_kv_cache for the cache).

No ntops counterpart (its attention, torch/scaled_dot_product_attention.py:10-108,
reads a cache of the query's type).  query (batch, query heads, tokens, head_dim)
attends the first lengths[b] tokens of sequence b (int32 or int64 (batch,);
None: the whole capacity; query head h reads cache head h // (query heads / cache
heads)).  With is_causal the last query row is the sequence's last token: row i
sees the keys up to lengths[b] - tokens + i.  A row that sees no key is 0; a
NaN value reaches the rows that see its token and no others.
Scales of the cache are not negative.
scale defaults to 1 / sqrt(head_dim).  float16, bfloat16 or float32 queries, head
dims up to 256; 16-bit queries of head dims that are multiples of 16 up to 128
run on the matrix cores."""

import math

import torch

from ntops_amd import _lib
from ntops_amd.torch.store_kv_cache import _checked_cache, _check_index
from ntops_amd.torch.utils import _DeviceGuard, _contiguous, _strides


def kv_cache_attention(
    query, key_cache, value_cache, key_scale, value_scale, lengths=None, is_causal=False, scale=None, *, block_size=64
):
    if _lib.fast is not None:
        r = _lib.fast.kv_cache_attention(
            query, key_cache, value_cache, key_scale, value_scale, lengths, is_causal, scale, block_size)
        if r is not None:
            return r
    what = "kv_cache_attention"
    b, hkv, c, d = _checked_cache(key_cache, value_cache, key_scale, value_scale, block_size, what)
    if query.dim() != 4 or query.shape[0] != b or query.shape[3] != d:
        raise RuntimeError(f"{what}: query {tuple(query.shape)} does not fit a cache of shape {(b, hkv, c, d)}")
    if query.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"{what}: unsupported dtype {query.dtype}")
    _, hq, sq, _ = query.shape
    if hkv == 0 or hq % hkv:
        raise RuntimeError(f"{what}: {hq} query heads are not a multiple of {hkv} cache heads")
    if lengths is not None:
        _check_index(lengths, b, "lengths", what)
    dev = _lib.require_cuda(query, key_cache, value_cache, key_scale, value_scale, lengths)
    if scale is None:
        scale = 1 / math.sqrt(d) if d else 1.0
    output = torch.empty(query.shape, dtype=query.dtype, device=dev)
    lib = _lib.load()
    dt = _lib.dtype_code(query.dtype)
    with _DeviceGuard(dev):
        if query.stride(3) != 1 and d > 1:
            query = _contiguous(query)
        for t in (key_cache, value_cache, key_scale, value_scale):
            if t.stride(-1) != 1 and t.shape[-1] > 1:
                raise RuntimeError(f"{what}: the last dim of a cache and its scales needs a unit stride")
        lengths = None if lengths is None else _contiguous(lengths)
        ws_bytes = lib.ntops_kv_cache_attention_workspace(dt, b, hq, hkv, sq, c, d)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        rc = lib.ntops_kv_cache_attention(
            dt, b, hq, hkv, sq, c, d, block_size, query.data_ptr(), _strides(query),
            key_cache.data_ptr(), _strides(key_cache), value_cache.data_ptr(), _strides(value_cache),
            key_scale.data_ptr(), _strides(key_scale), value_scale.data_ptr(), _strides(value_scale),
            None if lengths is None else lengths.data_ptr(), 0 if lengths is None else _lib.dtype_code(lengths.dtype),
            int(bool(is_causal)), float(scale), output.data_ptr(), _strides(output),
            None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream_of(output))
    _lib.check(rc, "ntops_amd.kv_cache_attention")
    return output
