"""mxfp4_mm -- the product of two MXFP4 matrices (see quantize_mxfp4) that share
their last dim, as a linear layer's activations and weight do:

    output = input @ mat2.T (+ bias)

No ntops counterpart (its products, torch/mm.py:7-18 and addmm.py:7-18, take 16
and 32 bits).  input (M, K) and mat2 (N, K) are codes with their scales; with
input_scale None, input is a float tensor (M, K) that is quantized first.  Sums
are fp32, bias (N,) of `dtype` is added in fp32, and the result is rounded once
to `dtype` (bfloat16, float16 or float32)."""

import torch

from ntops_amd import _lib
from ntops_amd.torch.dequantize_mxfp4 import _checked_pair
from ntops_amd.torch.quantize_mxfp4 import _DTYPES, _rows
from ntops_amd.torch.utils import _DeviceGuard, _cast_into, _contiguous


# (a tile's rows have to lie within 2^30 bytes)
_FARTHEST_ROWS = (1 << 30) // 257


def _code_rows(t):
    """t with rows that the kernels can read: unit stride, 16-byte aligned."""
    if t.stride(1) == 1 and 0 <= t.stride(0) <= _FARTHEST_ROWS and t.stride(0) % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return _cast_into(t, torch.empty(t.shape, dtype=t.dtype, device=t.device))


def _scale_rows(t):
    return t if t.stride(1) == 1 and 0 <= t.stride(0) <= _FARTHEST_ROWS else _contiguous(t)


def mxfp4_mm(input, input_scale, mat2, mat2_scale, bias=None, *, dtype=torch.bfloat16):
    if _lib.fast is not None:
        r = _lib.fast.mxfp4_mm(input, input_scale, mat2, mat2_scale, bias, dtype)
        if r is not None:
            return r
    if input.dim() != 2 or mat2.dim() != 2:
        raise RuntimeError("mxfp4_mm: expected 2-D tensors")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"mxfp4_mm: unsupported dtype {dtype}")
    blocks = _checked_pair(mat2, mat2_scale, "mxfp4_mm")
    dev = _lib.require_cuda(input, input_scale, mat2, mat2_scale, bias)
    m, n = input.shape[0], mat2.shape[0]
    if input_scale is None:
        if -(-input.shape[1] // 32) != blocks:
            raise RuntimeError(f"mxfp4_mm: rows of {input.shape[1]} values do not have mat2's {blocks} blocks of 32")
        if input.dtype not in _DTYPES:
            raise RuntimeError(f"quantize_mxfp4: unsupported dtype {input.dtype}")
    elif _checked_pair(input, input_scale, "mxfp4_mm") != blocks:
        raise RuntimeError(f"mxfp4_mm: {input_scale.shape[1]} and {blocks} blocks cannot be multiplied")
    if bias is not None and (bias.shape != (n,) or bias.dtype != dtype):
        raise RuntimeError(f"mxfp4_mm: expected a bias of shape ({n},) and dtype {dtype}, got {tuple(bias.shape)}, {bias.dtype}")

    output = torch.empty((m, n), dtype=dtype, device=dev)
    lib = _lib.load()
    with _DeviceGuard(dev):
        b, sb = _code_rows(mat2), _scale_rows(mat2_scale)
        bias = None if bias is None else _contiguous(bias)
        weight = b.data_ptr(), b.stride(0), sb.data_ptr(), sb.stride(0), None if bias is None else bias.data_ptr(), output.data_ptr(), n
        if input_scale is None:
            x, _, stride = _rows(input)
            k = x.shape[1]
            a = x.data_ptr(), stride
            ws_bytes = lib.ntops_mxfp4_linear_workspace(_lib.dtype_code(x.dtype), m, n, k, *a)
        else:
            x, sx = _code_rows(input), _scale_rows(input_scale)
            k = 32 * blocks
            a = x.data_ptr(), x.stride(0), sx.data_ptr(), sx.stride(0)
            ws_bytes = lib.ntops_mxfp4_mm_workspace(m, n, k)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
        rest = *a, *weight, None if ws is None else ws.data_ptr(), ws_bytes, _lib.stream_of(output)
        if input_scale is None:
            rc = lib.ntops_mxfp4_linear(_lib.dtype_code(x.dtype), _lib.dtype_code(dtype), m, n, k, *rest)
        else:
            rc = lib.ntops_mxfp4_mm(_lib.dtype_code(dtype), m, n, k, *rest)
    _lib.check(rc, "ntops_amd.mxfp4_mm")
    return output
