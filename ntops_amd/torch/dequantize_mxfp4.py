"""dequantize_mxfp4 -- the values of a tensor in MXFP4 (see quantize_mxfp4).

No ntops counterpart.  `size` is the length of the last dim (default: all that
the blocks hold); the values are rounded once to `dtype`."""

import torch

from ntops_amd import _lib
from ntops_amd.torch.utils import _DeviceGuard, _cast_into, _contiguous


def _checked_pair(codes, scales, what):
    """The number of blocks along the last dim of MXFP4 codes and scales."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise RuntimeError(f"{what}: expected uint8 codes and scales, got {codes.dtype} and {scales.dtype}")
    if (
        codes.dim() == 0
        or codes.dim() != scales.dim()
        or codes.shape[:-1] != scales.shape[:-1]
        or codes.shape[-1] != 16 * scales.shape[-1]
    ):
        raise RuntimeError(
            f"{what}: expected codes (..., 16 * blocks) and scales (..., blocks), got {tuple(codes.shape)} and "
            f"{tuple(scales.shape)}"
        )
    return scales.shape[-1]


def dequantize_mxfp4(codes, scales, size=None, *, dtype=torch.bfloat16):
    if _lib.fast is not None:
        r = _lib.fast.dequantize_mxfp4(codes, scales, size, dtype)
        if r is not None:
            return r
    blocks = _checked_pair(codes, scales, "dequantize_mxfp4")
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"dequantize_mxfp4: unsupported dtype {dtype}")
    if size is None:
        size = 32 * blocks
    elif -(-size // 32) != blocks or size < 0:
        raise RuntimeError(f"dequantize_mxfp4: a last dim of {size} does not have {blocks} blocks of 32")
    dev = _lib.require_cuda(codes, scales)
    output = torch.empty(codes.shape[:-1] + (size,), dtype=dtype, device=dev)
    lib = _lib.load()
    with _DeviceGuard(dev):
        codes, scales = _contiguous(codes), _contiguous(scales)
        if codes.data_ptr() % 4:
            codes = _cast_into(codes, torch.empty(codes.shape, dtype=codes.dtype, device=dev))
        rc = lib.ntops_dequantize_mxfp4(
            _lib.dtype_code(dtype), output.numel() // size if size else 0, size, codes.data_ptr(), 16 * blocks,
            scales.data_ptr(), blocks, output.data_ptr(), _lib.stream_of(output))
    _lib.check(rc, "ntops_amd.dequantize_mxfp4")
    return output
