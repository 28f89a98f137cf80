"""Linear layer in 8-bit floating point on HIP, gfx950: an e4m3 product with a scale for every 128
columns of a row and for every 128 x 128 values of the weight.

``fp8_gemm(q, scale, qweight, w_scale)`` multiplies rows quantized by ``quantize_fp8`` with a weight
quantized by ``slipstream_amd.quantized.quantize_weight_fp8`` (or stored so in a checkpoint). Each
block of 128 is summed by the matrix cores, times its scales, and added in fp32; the result is
rounded once to ``out_dtype``. For fp16 and fp32 a block's sum is in fp32; for bf16 it is the e4m3
instruction's, which drops what lies below 2^-13 of the largest of eight keys' products (2^-16 of the sum on
average over 128 normal products): below the half step of the result's type where large products do not cancel.
Ask for fp32 results where they do. The reference has no counterpart; the conventions are
those of ``w8a8_gemm``. Device tensors only.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device
from slipstream_amd.kernels.fp8_rows import FP8, blocks_of

# Workspace bytes the library asks for, by shape.
_WS_NEED: dict[tuple, int] = {}


def check_fp8_args(q: torch.Tensor, scale: torch.Tensor, qweight: torch.Tensor, w_scale: torch.Tensor,
                   bias: torch.Tensor | None) -> tuple[int, int]:
    """Shape and dtype checks; returns ``(out, in)``."""
    weight_shape, shape = qweight.shape, q.shape
    if len(weight_shape) != 2:
        raise ValueError(f"qweight must be 2-D [out, in], got {tuple(weight_shape)}")
    n, k = weight_shape
    if q.dtype != FP8 or qweight.dtype != FP8:
        raise ValueError(f"q and qweight must be float8_e4m3fn, got {q.dtype} and {qweight.dtype}")
    if scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise ValueError(f"scale and w_scale must be float32, got {scale.dtype} and {w_scale.dtype}")
    if not shape or shape[-1] != k:
        raise ValueError(f"q {tuple(shape)} does not end in the weight's {k} input features")
    blocks = blocks_of(k)
    if scale.shape != (*shape[:-1], blocks):
        raise ValueError(f"scale {tuple(scale.shape)} != {blocks} for each row of q {tuple(shape)}")
    if w_scale.shape != (blocks_of(n), blocks):
        raise ValueError(f"w_scale {tuple(w_scale.shape)} != [{blocks_of(n)}, {blocks}]: one for 128 x 128 values")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias {tuple(bias.shape)} != [out={n}]")
    return n, k


def _whole(t: torch.Tensor, stride: int) -> int:
    """Whether ``t``'s rows start on 16 bytes and are not further apart than the kernels reach."""
    return int(not (t.data_ptr() | stride) & 15 and stride <= 1 << 21)


def _workspace_need(device: torch.device, m: int, n: int, k: int, x_whole: int, w_whole: int, dtype: int) -> int:
    key = (device.index, m, n, k, x_whole, w_whole, dtype)
    need = _WS_NEED.get(key)
    if need is None:
        out = _ffi.ctypes.c_int64(0)
        with torch.cuda.device(device):
            status = _ffi.lib().ss_fp8_workspace_size(m, n, k, x_whole, w_whole, dtype,
                                                        _ffi.ctypes.byref(out))
        _ffi.check(status, "fp8 workspace")
        if len(_WS_NEED) > 4096:  # many distinct shapes: start over
            _WS_NEED.clear()
        need = _WS_NEED[key] = int(out.value)
    return need


def _scale_rows(scale: torch.Tensor, m: int) -> torch.Tensor:
    """``scale [..., blocks]`` as ``[m, blocks]``, without a copy where its rows are evenly apart."""
    if scale.ndim == 2:
        return scale
    blocks = scale.shape[-1]
    by_block = scale.movedim(-1, 0)
    return by_block.reshape(blocks, m).t() if by_block.is_contiguous() else scale.reshape(m, blocks)


def fp8_gemm(q: torch.Tensor, scale: torch.Tensor, qweight: torch.Tensor, w_scale: torch.Tensor,
             bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dequant(q) @ dequant(qweight).T (+ bias)`` in ``out_dtype``: ``q [..., in]`` float8_e4m3fn,
    ``scale [..., ceil(in / 128)]`` fp32 of any layout, ``qweight [out, in]`` float8_e4m3fn, ``w_scale
    [ceil(out / 128), ceil(in / 128)]`` fp32, ``bias [out]`` of any float dtype -> ``[..., out]``."""
    n, k = check_fp8_args(q, scale, qweight, w_scale, bias)
    dtype = _ffi.dtype_code(out_dtype)
    bias_dtype = _ffi.dtype_code(bias.dtype) if bias is not None else 0
    out = q.new_empty((*q.shape[:-1], n), dtype=out_dtype)
    if out.numel() == 0:
        return out
    if bias is None:
        require_device("fp8_gemm", q, scale, qweight, w_scale)
    else:
        require_device("fp8_gemm", q, scale, qweight, w_scale, bias)
        bias = bias.contiguous()
    m = out.numel() // n
    q_stride = w_stride = k
    if not q.is_contiguous():
        q = q.reshape(m, k)
        if k and (q.stride(1) != 1 or (m > 1 and q.stride(0) < k)):
            q = q.contiguous()
        q_stride = q.stride(0)
    if not qweight.is_contiguous():
        if k and (qweight.stride(1) != 1 or (n > 1 and qweight.stride(0) < k)):
            qweight = qweight.contiguous()
        w_stride = qweight.stride(0)
    scale = _scale_rows(scale, m)
    need = _workspace_need(q.device, m, n, k, _whole(q, q_stride), _whole(qweight, w_stride), dtype)
    # of this call alone: nothing is shared between streams, or between captured graphs
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    status = launch(q.device, _ffi.lib().ss_fp8_gemm, q.data_ptr(), scale.data_ptr(), qweight.data_ptr(),
                    w_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k, q_stride,
                    w_stride, n, _ffi.i64x2(*scale.stride()), _ffi.i64x2(*w_scale.stride()), dtype, bias_dtype,
                    None if ws is None else ws.data_ptr(), need)
    _ffi.check(status, "fp8_gemm")
    return out
