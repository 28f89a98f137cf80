"""W8A8 linear on HIP, gfx950: an int8 product with a scale for each token and each channel.

``w8a8_gemm(q, scale, qweight, w_scale)`` multiplies rows quantized by ``quantize_int8``,
``fused_rmsnorm_int8`` or ``fused_swiglu_int8`` with a weight quantized per output channel
(``slipstream_amd.quantized.quantize_weight_int8``). The integer sum is exact (int32), so a
result does not depend on the batch around it nor on the kernel that ran: it is rounded by
the scales in fp32 and once to ``out_dtype``. The reference has no counterpart; the
conventions are those of ``w4a16_gemm``. Device tensors only.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device

# Workspace bytes the library asks for, by shape.
_WS_NEED: dict[tuple, int] = {}


def check_w8a8_args(q: torch.Tensor, scale: torch.Tensor, qweight: torch.Tensor, w_scale: torch.Tensor,
                    bias: torch.Tensor | None) -> tuple[int, int]:
    """Shape and dtype checks; returns ``(out, in)``."""
    weight_shape, shape = qweight.shape, q.shape
    if len(weight_shape) != 2:
        raise ValueError(f"qweight must be 2-D [out, in], got {tuple(weight_shape)}")
    n, k = weight_shape
    if q.dtype != torch.int8 or qweight.dtype != torch.int8:
        raise ValueError(f"q and qweight must be int8, got {q.dtype} and {qweight.dtype}")
    if scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise ValueError(f"scale and w_scale must be float32, got {scale.dtype} and {w_scale.dtype}")
    if not shape or shape[-1] != k:
        raise ValueError(f"q {tuple(shape)} does not end in the weight's {k} input features")
    if scale.shape != shape[:-1]:
        raise ValueError(f"scale {tuple(scale.shape)} != one for each row of q {tuple(shape)}")
    if w_scale.shape != (n,):
        raise ValueError(f"w_scale {tuple(w_scale.shape)} != [out={n}]")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias {tuple(bias.shape)} != [out={n}]")
    return n, k


def _whole(t: torch.Tensor, stride: int) -> int:
    """Whether ``t``'s rows start on 16 bytes and are not further apart than the kernels reach."""
    return int(not (t.data_ptr() | stride) & 15 and stride <= 1 << 21)


def _workspace_need(device: torch.device, m: int, n: int, k: int, x_whole: int, w_whole: int) -> int:
    key = (device.index, m, n, k, x_whole, w_whole)
    need = _WS_NEED.get(key)
    if need is None:
        out = _ffi.ctypes.c_int64(0)
        with torch.cuda.device(device):
            status = _ffi.lib().ss_w8a8_workspace_size(m, n, k, x_whole, w_whole, _ffi.ctypes.byref(out))
        _ffi.check(status, "w8a8 workspace")
        if len(_WS_NEED) > 4096:  # many distinct shapes: start over
            _WS_NEED.clear()
        need = _WS_NEED[key] = int(out.value)
    return need


def w8a8_gemm(q: torch.Tensor, scale: torch.Tensor, qweight: torch.Tensor, w_scale: torch.Tensor,
              bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(q * scale[..., None]) @ (qweight * w_scale[:, None]).T (+ bias)`` in ``out_dtype``:
    ``q [..., in]`` int8, ``scale [...]`` fp32, ``qweight [out, in]`` int8, ``w_scale [out]``
    fp32, ``bias [out]`` of any float dtype -> ``[..., out]``."""
    n, k = check_w8a8_args(q, scale, qweight, w_scale, bias)
    dtype = _ffi.dtype_code(out_dtype)
    bias_dtype = _ffi.dtype_code(bias.dtype) if bias is not None else 0
    out = q.new_empty((*q.shape[:-1], n), dtype=out_dtype)
    if out.numel() == 0:
        return out
    if bias is None:
        require_device("w8a8_gemm", q, scale, qweight, w_scale)
    else:
        require_device("w8a8_gemm", q, scale, qweight, w_scale, bias)
        bias = bias.contiguous()
    m = scale.numel()
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
    scale, w_scale = scale.contiguous(), w_scale.contiguous()
    need = _workspace_need(q.device, m, n, k, _whole(q, q_stride), _whole(qweight, w_stride))
    # of this call alone: nothing is shared between streams, or between captured graphs
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    status = launch(q.device, _ffi.lib().ss_w8a8_gemm, q.data_ptr(), scale.data_ptr(), qweight.data_ptr(),
                    w_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k, q_stride,
                    w_stride, n, dtype, bias_dtype, None if ws is None else ws.data_ptr(), need)
    _ffi.check(status, "w8a8_gemm")
    return out
