"""multi_axis_rotary_position_embedding_qk -- rotary positions with several axes (of
an image or a video: time, height and width) on the query and key of one attention
layer, in a single launch.

No ntops counterpart (torch/rotary_position_embedding.py:7-29 rotates a whole head by
one position, the token's place).  q (batch, seq, q_heads, dim) and k (batch, seq,
k_heads, dim); positions (axes, batch, seq) in int32 or int64, expanded dims as they
are.  `sections` divides the dim / 2 pairs of a head: section s holds that many pairs
in order, and belongs to axis s % axes -- (16, 24, 24) for three blocks of pairs,
(1,) * 64 for axes in turn.  A pair's angle is that of its axis' position: sin_table
and cos_table (positions, dim / 2), or (positions, dim) with each element's own
column, in float32 or the tensors' type.  Pairs are elements (2 i, 2 i + 1), or with
interleaved=False (i, i + dim / 2).

Computed in fp32 and rounded once.  A pair whose position lies outside of the tables
is NaN (positions are read on the device).  Returns (q_out, k_out); inplace=True
rotates q and k in place, where each element is one of its own: tensors that share
elements with each other or with themselves are refused."""

import operator

import torch

from ntops_amd import _lib
from ntops_amd.torch.utils import _DeviceGuard, _contiguous, _strides, _to_dtype


def _reaches(target, terms):
    """Whether `target` is the sum of step * n over the (step, most) of `terms`, for some n of 0 .. most
    each.  Largest steps first, which leave few n where strides are those of nested dims; True
    where 10000 trials do not tell."""
    most_of = {}
    for step, most in terms:
        if step and most:
            most_of[step] = most_of.get(step, 0) + most
    steps = sorted(most_of.items(), reverse=True)
    rest = [0]
    for step, most in reversed(steps):
        rest.append(rest[-1] + step * most)
    rest.reverse()
    todo = [(0, target)]
    for _ in range(10000):
        if not todo:
            return False
        i, left = todo.pop()
        if left == 0:
            return True
        if left < 0 or left > rest[i]:
            continue
        step, most = steps[i]
        first, last = max(0, -((rest[i + 1] - left) // step)), min(most, left // step)
        if last - first > 10000:
            return True
        todo += [(i + 1, left - n * step) for n in range(first, last + 1)]
    return True


def _dims(x):
    return [(s, n - 1) for s, n in zip(x.stride(), x.shape) if n > 1]


def _meets_itself(x):
    """Whether two elements of x are the same memory."""
    if not x.numel():
        return False
    end = 1
    for step, most in sorted(_dims(x)):
        if step < end:
            break
        end += step * most
    else:
        return False  # each dim's step passes all that the smaller ones reach
    # index vectors that differ first in dim i, by n + 1, and by -most .. most behind it
    dims = _dims(x)
    return any(
        step == 0 or _reaches(sum(s * m for s, m in dims[i + 1 :]) - step, [(step, most - 1)] + [(s, 2 * m) for s, m in dims[i + 1 :]])
        for i, (step, most) in enumerate(dims))


def _meet(q, k):
    """Whether an element of q and one of k are the same memory (both of one type)."""
    if not q.numel() or not k.numel():
        return False
    size = q.element_size()
    apart = k.data_ptr() - q.data_ptr()
    q_end, k_end = (sum(s * m for s, m in _dims(x)) for x in (q, k))
    if apart > q_end * size or -apart > k_end * size:
        return False
    # q's index vector, and k's counted from its last element
    return apart % size != 0 or _reaches(apart // size + k_end, _dims(q) + _dims(k))


def multi_axis_rotary_position_embedding_qk(q, k, sin_table, cos_table, positions, sections, interleaved=True, inplace=False):
    if _lib.fast is not None:
        r = _lib.fast.rope_axes_qk(q, k, sin_table, cos_table, positions, sections, interleaved, inplace)
        if r is not None:
            return r
    what = "multi_axis_rotary_position_embedding_qk"
    if q.dim() != 4 or k.dim() != 4:
        raise RuntimeError(f"{what}: q and k must be (batch, seq, heads, dim)")
    batch, seq, _, dim = q.shape
    if k.shape[0] != batch or k.shape[1] != seq or k.shape[3] != dim:
        raise RuntimeError(f"{what}: q and k differ in batch, seq or dim")
    if k.dtype != q.dtype or q.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"{what}: expected one of float32, float16 and bfloat16, got {q.dtype} and {k.dtype}")
    if dim % 2 != 0:
        raise RuntimeError("The embedding dimension must be even.")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 3 or positions.shape[1:] != (batch, seq) or positions.shape[0] < 1:
        raise RuntimeError(f"{what}: expected positions of shape (axes, {batch}, {seq}) in int32 or int64, got {tuple(positions.shape)}, {positions.dtype}")
    sections = [operator.index(n) for n in sections]
    if min(sections, default=-1) < 0 or sum(sections) != dim // 2:
        raise RuntimeError(f"{what}: sections {sections} do not add up to {dim // 2} pairs")
    if sin_table.dim() != 2 or sin_table.shape != cos_table.shape or sin_table.shape[1] not in (dim // 2, dim):
        raise RuntimeError(
            f"{what}: the tables must both be (positions, {dim // 2}) or (positions, {dim}), got {tuple(sin_table.shape)} and {tuple(cos_table.shape)}")
    if inplace and (_meets_itself(q) or _meets_itself(k)):
        raise RuntimeError(f"{what}: elements that share memory cannot be rotated in place")
    if inplace and _meet(q, k):
        raise RuntimeError(f"{what}: q and k share elements, which would be rotated twice in place")
    dev = _lib.require_cuda(q, k, sin_table, cos_table, positions)
    lib = _lib.load()
    with _DeviceGuard(dev):
        q_out = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=dev)
        k_out = k if inplace else torch.empty(k.shape, dtype=k.dtype, device=dev)
        tables = [sin_table, cos_table]
        if sin_table.dtype != cos_table.dtype or sin_table.dtype not in (torch.float32, q.dtype):
            tables = [_to_dtype(t, torch.float32) for t in tables]
        sin_table, cos_table = (t if t.stride(1) == 1 or t.shape[1] <= 1 else _contiguous(t) for t in tables)
        rc = lib.ntops_rope_axes_qk(
            _lib.dtype_code(q.dtype), batch, seq, q.shape[2], k.shape[2], dim,
            q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), _lib.dtype_code(sin_table.dtype),
            sin_table.data_ptr(), sin_table.stride(0), cos_table.data_ptr(), cos_table.stride(0),
            sin_table.shape[0], sin_table.shape[1], positions.shape[0], positions.data_ptr(),
            _lib.dtype_code(positions.dtype), _strides(positions), len(sections), _lib.i64_array(sections),
            1 if interleaved else 0, q_out.data_ptr(), _strides(q_out), k_out.data_ptr(), _strides(k_out),
            _lib.stream_of(q_out))
    _lib.check(rc, f"ntops_amd.{what}")
    return q_out, k_out
