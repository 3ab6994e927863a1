"""quantize_mxfp4 -- microscaled 4-bit floating point (OCP MXFP4) of a tensor.

No ntops counterpart.  The last dim is cut into blocks of 32 (the last one
padded with zeros).  A block's scale is 2^e, e = max(-127, floor(log2(max |x|))
- 2), and its values are x / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3,
4, 6 (ties to the even code) and cut at 6.  Returns

  codes   uint8 (..., 16 * blocks): two 4-bit codes a byte, the first in the low
          half; sign in bit 3
  scales  uint8 (..., blocks): the bytes e + 127

A block with a NaN or an infinity has the scale 255 and stands for NaN."""

import torch

from ntops_amd import _lib
from ntops_amd.torch.utils import _DeviceGuard, _contiguous

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _rows(t):
    """(tensor, rows, row stride): t's last dim as rows of a 2-D layout, a
    row-major copy where it is none."""
    shape, stride = t.shape, t.stride()
    cols = shape[-1]
    rows = t.numel() // cols if cols else 0
    if t.dim() == 2 and (stride[1] == 1 or cols == 1) and stride[0] >= 0:
        return t, rows, stride[0]
    return _contiguous(t), rows, cols


def quantize_mxfp4(input):
    if _lib.fast is not None:
        r = _lib.fast.quantize_mxfp4(input)
        if r is not None:
            return r
    if input.dim() == 0:
        raise RuntimeError("quantize_mxfp4: expected a tensor of at least one dim")
    if input.dtype not in _DTYPES:
        raise RuntimeError(f"quantize_mxfp4: unsupported dtype {input.dtype}")
    dev = _lib.require_cuda(input)
    cols = input.shape[-1]
    blocks = -(-cols // 32)
    codes = torch.empty(input.shape[:-1] + (16 * blocks,), dtype=torch.uint8, device=dev)
    scales = torch.empty(input.shape[:-1] + (blocks,), dtype=torch.uint8, device=dev)
    lib = _lib.load()
    with _DeviceGuard(dev):
        x, rows, stride = _rows(input)
        rc = lib.ntops_quantize_mxfp4(
            _lib.dtype_code(x.dtype), rows, cols, x.data_ptr(), stride, codes.data_ptr(), scales.data_ptr(),
            _lib.stream_of(codes))
    _lib.check(rc, "ntops_amd.quantize_mxfp4")
    return codes, scales
