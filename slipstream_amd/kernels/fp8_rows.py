"""Rows quantized to 8-bit floating point with a scale for every 128 columns (HIP, gfx950): the
inputs of ``fp8_gemm``.

A block ``x`` of a row becomes ``scale = max|x| / 448`` and ``q = e4m3(x * 448 / max|x|)``, the exact
quotient rounded to the nearest, half to even. A block of zeros (or below 5.3e-36) has scale 0; a
block with a NaN or an infinity has zeros and scale NaN. The reference has no counterpart; the
conventions are those of ``quantize_int8``. Device tensors only.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device
from slipstream_amd.kernels.norm_act import _rows

FP8 = torch.float8_e4m3fn
BLOCK = 128  # columns (of a weight: rows too) that share a scale


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` -> ``(q float8_e4m3fn [..., K], scale fp32 [..., ceil(K / 128)])``; ``scale`` is
    laid out block by block (all rows' first scales, then all rows' second ones, ...), as the product
    reads it fastest."""
    shape = x.shape
    if not shape:
        raise ValueError("rows need at least one dimension")
    dtype = _ffi.dtype_code(x.dtype)
    cols = shape[-1]
    q = x.new_empty(shape, dtype=FP8)
    by_block = x.new_empty((blocks_of(cols), *shape[:-1]), dtype=torch.float32)
    scale = by_block.t() if x.ndim == 2 else by_block.movedim(0, -1)
    if q.numel() == 0:
        return q, scale
    require_device("quantize_fp8", x)
    rows = q.numel() // cols
    x2, xs = (x, cols) if x.is_contiguous() else _rows(x, cols)
    status = launch(x.device, _ffi.lib().ss_quantize_fp8, x2.data_ptr(), q.data_ptr(), by_block.data_ptr(), rows, cols,
                    xs, rows, dtype)
    _ffi.check(status, "quantize_fp8")
    return q, scale
