"""store_kv_cache -- new keys and values into a cache held in 8 bits.

No ntops counterpart: its cache (kernels/scaled_dot_product_attention.py:139-140)
is of the query's type.  The cache of a layer is four tensors of the caller's:

  key_cache, value_cache   float8_e4m3fn (batch, heads, capacity, head_dim)
  key_scale, value_scale   float32 (batch, heads, ceil(capacity / block_size))

A token's values are its codes times the scale of its block of `block_size` (a
power of two of 16 to 2^24) tokens.  key and value (batch, heads, tokens,
head_dim; float32, float16 or bfloat16) go to `positions` and on: an int, or an
int32 / int64 tensor (batch,).  With `lengths` (batch,) only each sequence's
first lengths[b] tokens are stored.  Tokens outside of the cache are dropped.

A block's scale is the least power of two, 2^-126 at least, under which its
largest finite value is at most 448; what is not finite is stored as NaN.  Tokens
that start inside a block keep the larger of its scale and theirs; where that
raises it, the block's earlier tokens are rounded again.  What the cache holds
behind the new tokens stays as it is, and means nothing in the rest of their last
block: a sequence grows at its end, or is cut and grows from there."""

import operator

import torch

from ntops_amd import _lib
from ntops_amd.torch.utils import _DeviceGuard, _contiguous, _strides


def _checked_cache(key_cache, value_cache, key_scale, value_scale, block_size, what):
    """The cache's shape (batch, heads, capacity, head_dim)."""
    if not 16 <= block_size <= 1 << 24 or block_size & (block_size - 1):
        raise RuntimeError(f"{what}: block_size must be a power of two of 16 to 2^24, got {block_size}")
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        raise RuntimeError(f"{what}: expected two 4-D caches of one shape, got {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
    if key_cache.dtype != torch.float8_e4m3fn or value_cache.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"{what}: expected float8_e4m3fn caches, got {key_cache.dtype} and {value_cache.dtype}")
    b, h, c, _ = key_cache.shape
    want = (b, h, -(-c // block_size))
    for s in (key_scale, value_scale):
        if s.dtype != torch.float32 or s.shape != want:
            raise RuntimeError(f"{what}: expected float32 scales of shape {want}, got {s.dtype}, {tuple(s.shape)}")
    return key_cache.shape


def _check_index(t, batch, name, what):
    """Refuses an index vector that is not one integer per sequence."""
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (batch,):
        raise RuntimeError(f"{what}: expected {name} of shape ({batch},) in int32 or int64, got {tuple(t.shape)}, {t.dtype}")


def store_kv_cache(key, value, key_cache, value_cache, key_scale, value_scale, positions, lengths=None, *, block_size=64):
    if _lib.fast is not None and _lib.fast.store_kv_cache(
        key, value, key_cache, value_cache, key_scale, value_scale, positions, lengths, block_size
    ):
        return
    what = "store_kv_cache"
    b, h, c, d = _checked_cache(key_cache, value_cache, key_scale, value_scale, block_size, what)
    if key.dim() != 4 or key.shape != value.shape or key.shape[:2] != (b, h) or key.shape[3] != d:
        raise RuntimeError(f"{what}: key {tuple(key.shape)} and value {tuple(value.shape)} do not fit a cache of shape {(b, h, c, d)}")
    if key.dtype != value.dtype or key.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"{what}: unsupported dtypes {key.dtype} and {value.dtype}")
    tensors = [key, value, key_cache, value_cache, key_scale, value_scale, lengths]
    at = 0
    if isinstance(positions, torch.Tensor):
        _check_index(positions, b, "positions", what)
        tensors.append(positions)
    else:
        at, positions = max(-(1 << 62), min(1 << 62, operator.index(positions))), None
    if lengths is not None:
        _check_index(lengths, b, "lengths", what)
    for t in (key_cache, value_cache, key_scale, value_scale):
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise RuntimeError(f"{what}: the cache's tokens share memory (a stride is 0)")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise RuntimeError(f"{what}: the last dim of a cache and its scales needs a unit stride")
    dev = _lib.require_cuda(*tensors)
    lib = _lib.load()
    with _DeviceGuard(dev):
        key, value = (x if x.stride(3) == 1 or d <= 1 else _contiguous(x) for x in (key, value))
        positions, lengths = (None if t is None else _contiguous(t) for t in (positions, lengths))
        rc = lib.ntops_store_kv_cache(
            _lib.dtype_code(key.dtype), b, h, key.shape[2], d, c, block_size,
            key.data_ptr(), _strides(key), value.data_ptr(), _strides(value),
            key_cache.data_ptr(), _strides(key_cache), value_cache.data_ptr(), _strides(value_cache),
            key_scale.data_ptr(), _strides(key_scale), value_scale.data_ptr(), _strides(value_scale),
            None if positions is None else positions.data_ptr(), 0 if positions is None else _lib.dtype_code(positions.dtype), at,
            None if lengths is None else lengths.data_ptr(), 0 if lengths is None else _lib.dtype_code(lengths.dtype),
            _lib.stream_of(key_cache))
    _lib.check(rc, "ntops_amd.store_kv_cache")
