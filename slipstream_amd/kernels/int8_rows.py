"""Rows quantized to int8 with a scale each (HIP, gfx950): the inputs of ``w8a8_gemm``.

``quantize_int8`` takes rows as they are, ``fused_rmsnorm_int8`` behind the RMS norm with the
residual's addition, ``fused_swiglu_int8`` behind SwiGLU; the names and arguments follow
``fused_rmsnorm`` and ``fused_swiglu``. A row ``y`` becomes ``q = rint(y * 127 / max|y|)`` and
``scale = max|y| / 127``. Everything between the inputs and ``q`` is fp32: unlike the 16-bit
ops, nothing is rounded to the inputs' type on the way, except the residual sum that is
returned. The norm's ``q`` is the exact quotient's (of ``s * weight`` in fp32); the others round
``1 / max|y|``, its product with 127 and that with ``y`` to fp32. A row of zeros (or of ``y``, for
the norm ``s * weight``, below 1.5e-36) has scale 0, whatever the norm's eps; a row with a NaN or
an infinity (for the norm in ``s * weight``) has zeros and scale NaN. Device tensors only.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device
from slipstream_amd.kernels.norm_act import _rows


def _outputs(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    shape = x.shape
    if not shape:
        raise ValueError("rows need at least one dimension")
    make = x.new_empty if shape[-1] else x.new_zeros
    return _like(x, torch.int8), make(shape[:-1], dtype=torch.float32)


def _like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of ``x``'s shape (``empty_like`` is the cheaper call)."""
    return torch.empty_like(x, dtype=dtype) if x.is_contiguous() else x.new_empty(x.shape, dtype=dtype)


def _flat(x: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """``x`` itself where its rows follow each other, else ``_rows``; and the row stride."""
    return (x, cols) if x.is_contiguous() else _rows(x, cols)


def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` -> ``(q int8 [..., K], scale fp32 [...])`` with ``x ~ q * scale[..., None]``."""
    dtype = _ffi.dtype_code(x.dtype)
    q, scale = _outputs(x)
    if q.numel() == 0:
        return q, scale
    require_device("quantize_int8", x)
    cols = x.shape[-1]
    x2, xs = _flat(x, cols)
    status = launch(x.device, _ffi.lib().ss_quantize_int8, x2.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(),
                    cols, xs, dtype)
    _ffi.check(status, "quantize_int8")
    return q, scale


def fused_rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``rms(x) * w``, or ``rms(x + residual) * w`` when ``residual`` is set, in int8:
    ``(q, scale, s)``. ``s`` is ``x + residual`` in ``x``'s dtype, the next residual, a new
    tensor (None without a residual)."""
    q, scale = _outputs(x)
    cols = x.shape[-1]
    if weight.numel() != cols:
        raise ValueError(f"weight numel {weight.numel()} != hidden {cols}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} != x {tuple(x.shape)}")
    if weight.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        dtypes = {x.dtype, weight.dtype} | ({residual.dtype} if residual is not None else set())
        raise ValueError(f"x, weight and residual must share a dtype, got {sorted(map(str, dtypes))}")
    dtype = _ffi.dtype_code(x.dtype)
    s = _like(x, x.dtype) if residual is not None else None
    if q.numel() == 0:
        return q, scale, s
    x2, xs = _flat(x, cols)
    w = weight.contiguous()
    if residual is None:
        require_device("fused_rmsnorm_int8", x, weight)
        r_ptr, rs, s_ptr = None, 0, None
    else:
        require_device("fused_rmsnorm_int8", x, weight, residual)
        r2, rs = _flat(residual, cols)
        r_ptr, s_ptr = r2.data_ptr(), s.data_ptr()
    status = launch(x.device, _ffi.lib().ss_rmsnorm_int8, x2.data_ptr(), r_ptr, w.data_ptr(), q.data_ptr(),
                    scale.data_ptr(), s_ptr, scale.numel(), cols, xs, rs, eps, dtype)
    _ffi.check(status, "fused_rmsnorm_int8")
    return q, scale, s


def fused_swiglu_int8(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``silu(gate) * up`` in int8: ``(q, scale)``."""
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate/up must share shape and dtype")
    dtype = _ffi.dtype_code(gate.dtype)
    q, scale = _outputs(gate)
    if q.numel() == 0:
        return q, scale
    require_device("fused_swiglu_int8", gate, up)
    cols = gate.shape[-1]
    g2, gs = _flat(gate, cols)
    u2, us = _flat(up, cols)
    status = launch(gate.device, _ffi.lib().ss_swiglu_int8, g2.data_ptr(), u2.data_ptr(), q.data_ptr(),
                    scale.data_ptr(), scale.numel(), cols, gs, us, dtype)
    _ffi.check(status, "fused_swiglu_int8")
    return q, scale
