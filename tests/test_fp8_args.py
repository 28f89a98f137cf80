"""The 8-bit floating point path's host checks (shapes, dtypes, devices, the C ABI's own), the weight
quantizer, which is torch on any device, and the oracle (no GPU needed)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8 as ora
from slipstream_amd import _ffi
from slipstream_amd.kernels import fp8_gemm, quantize_fp8
from slipstream_amd.kernels.fp8_rows import FP8
from slipstream_amd.quantized import FP8Linear, FP8MLP, quantize_weight_fp8

FAKE = 1 << 20  # a 16-byte aligned address that no refused call reads


def _fp8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(FP8)


def _gemm_args(**change):
    a = {"q": _fp8(2, 3, 200), "scale": torch.zeros(2, 3, 2), "qweight": _fp8(130, 200), "w_scale": torch.zeros(2, 2),
         "bias": None}
    return {**a, **change}


@pytest.mark.parametrize("change,match", [
    ({"q": torch.zeros(2, 3, 200)}, "must be float8_e4m3fn"),
    ({"q": torch.zeros(2, 3, 200, dtype=torch.int8)}, "must be float8_e4m3fn"),
    ({"qweight": torch.zeros(130, 200, dtype=torch.uint8).view(torch.float8_e5m2)}, "must be float8_e4m3fn"),
    ({"qweight": _fp8(130, 2, 100)}, "2-D"),
    ({"qweight": _fp8(130, 199)}, "199 input features"),
    ({"scale": torch.zeros(2, 3, 2, dtype=torch.bfloat16)}, "float32"),
    ({"w_scale": torch.zeros(2, 2, dtype=torch.float64)}, "float32"),
    ({"scale": torch.zeros(2, 3, 1)}, "2 for each row"),
    ({"scale": torch.zeros(2, 3)}, "2 for each row"),
    ({"w_scale": torch.zeros(1, 2)}, "w_scale"),
    ({"w_scale": torch.zeros(130, 2)}, "w_scale"),
    ({"bias": torch.zeros(1)}, "bias"),
])
def test_gemm_refuses_shapes_and_dtypes(change, match):
    with pytest.raises(ValueError, match=match):
        fp8_gemm(**_gemm_args(**change))


def test_other_types_and_devices_are_refused():
    with pytest.raises(_ffi.KernelError, match="not supported"):
        fp8_gemm(**_gemm_args(), out_dtype=torch.float64)
    with pytest.raises(_ffi.KernelError, match="not supported"):
        fp8_gemm(**_gemm_args(bias=torch.zeros(130, dtype=torch.int32)))
    with pytest.raises(_ffi.KernelError, match="not supported"):
        quantize_fp8(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="HIP devices only"):
        fp8_gemm(**_gemm_args())
    with pytest.raises(RuntimeError, match="HIP devices only"):
        quantize_fp8(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="dimension"):
        quantize_fp8(torch.zeros(()))


def test_empty_calls_compute_nothing():
    """No tokens, no channels, no columns: the shapes come back, without a device."""
    assert fp8_gemm(**_gemm_args(q=_fp8(0, 200), scale=torch.zeros(0, 2))).shape == (0, 130)
    assert fp8_gemm(**_gemm_args(qweight=_fp8(0, 200), w_scale=torch.zeros(0, 2))).shape == (2, 3, 0)
    for shape, blocks in (((0, 5, 300), (0, 5, 3)), ((4, 0), (4, 0))):
        q, scale = quantize_fp8(torch.zeros(shape))
        assert q.shape == shape and q.dtype == FP8 and scale.shape == blocks


def test_c_entries_refuse_before_any_launch():
    lib = _ffi.lib()
    two = _ffi.i64x2(1, 1)
    gemm = lambda m, n, k, **c: lib.ss_fp8_gemm(  # noqa: E731
        c.get("x", FAKE), FAKE, FAKE, FAKE, c.get("bias"), FAKE, m, n, k, c.get("xs", k), c.get("ws", k), c.get("os", n),
        two, two, c.get("dtype", _ffi.SS_DTYPE_BF16), c.get("bias_dtype", 0), None, 0, None)
    assert gemm(-1, 8, 8) == _ffi.SS_ERR_INVALID
    assert gemm(2, 8, 8, x=None) == _ffi.SS_ERR_INVALID and b"null" in lib.ss_last_error()
    assert gemm(2, 8, 8, xs=7) == _ffi.SS_ERR_INVALID and b"shorter" in lib.ss_last_error()
    assert gemm(2, 8, 8, ws=7) == _ffi.SS_ERR_INVALID
    assert gemm(2, 8, 8, os=7) == _ffi.SS_ERR_INVALID
    assert gemm(2, 8, 8, dtype=9) == _ffi.SS_ERR_UNSUPPORTED
    assert gemm(2, 8, 8, bias=FAKE, bias_dtype=9) == _ffi.SS_ERR_UNSUPPORTED
    assert gemm(2, 8, 1 << 30) == _ffi.SS_ERR_UNSUPPORTED
    assert gemm(0, 8, 8, x=None) == _ffi.SS_OK
    rows = lambda r, c, **o: lib.ss_quantize_fp8(  # noqa: E731
        o.get("x", FAKE), FAKE, FAKE, r, c, o.get("xs", c), o.get("ss", r), o.get("dtype", 1), None)
    assert rows(-1, 8) == _ffi.SS_ERR_INVALID
    assert rows(2, 8, x=None) == _ffi.SS_ERR_INVALID
    assert rows(2, 8, xs=7) == _ffi.SS_ERR_INVALID
    assert rows(2, 8, ss=1) == _ffi.SS_ERR_INVALID
    assert rows(2, 8, dtype=5) == _ffi.SS_ERR_UNSUPPORTED
    assert rows(2, 1 << 30) == _ffi.SS_ERR_UNSUPPORTED
    assert rows(1 << 40, 256) == _ffi.SS_ERR_UNSUPPORTED
    assert rows(0, 8, x=None) == _ffi.SS_OK
    need = ctypes.c_int64(-1)
    assert lib.ss_fp8_workspace_size(4, 8, -1, 1, 1, 1, ctypes.byref(need)) == _ffi.SS_ERR_INVALID
    assert lib.ss_fp8_workspace_size(4, 8, 8, 1, 1, 1, None) == _ffi.SS_ERR_INVALID


def test_oracle_rounds_as_the_type_does():
    """Every e4m3 value is kept, every halfway point goes to the even neighbour, and what lies a little to
    its sides to the nearer one: against the type's own list of values."""
    codes = torch.arange(256, dtype=torch.uint8).view(FP8).double()
    values = np.unique(codes[codes.isfinite()].numpy())
    assert len(values) == 253 and np.array_equal(ora.e4m3(values), values)
    half = (values[1:] + values[:-1]) / 2
    even = np.array([int(v) % 2 == 0 for v in torch.from_numpy(values).to(FP8).view(torch.uint8)])
    assert np.array_equal(ora.e4m3(half), np.where(even[:-1], values[:-1], values[1:]))
    assert np.array_equal(ora.e4m3(half + 1e-9), values[1:]) and np.array_equal(ora.e4m3(half - 1e-9), values[:-1])


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 300), (300, 127)])
def test_weight_quantizer(n, k):
    gen = torch.Generator().manual_seed(n * 1000 + k)
    w = (torch.randn(n, k, generator=gen) * 0.1).to(torch.bfloat16)
    w[:128, 128:256] = 0
    q, scales = quantize_weight_fp8(w)
    assert q.dtype == FP8 and q.shape == w.shape and scales.shape == (-(-n // 128), -(-k // 128))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = w[128 * i : 128 * i + 128, 128 * j : 128 * j + 128].double().numpy()
            top = np.abs(part).max()
            got = q[128 * i : 128 * i + 128, 128 * j : 128 * j + 128].double().numpy()
            if top == 0:
                assert scales[i, j] == 0 and not got.any()
                continue
            assert scales[i, j] == np.float32(top) / np.float32(448)
            assert np.array_equal(got, ora.e4m3(part * 448 / top))


def test_weight_quantizer_refuses():
    with pytest.raises(ValueError, match="2-D"):
        quantize_weight_fp8(torch.zeros(3))
    with pytest.raises(ValueError, match="NaN"):
        quantize_weight_fp8(torch.full((2, 2), float("nan")))


def test_linear_keeps_its_types_and_refuses_others():
    lin = FP8Linear.from_linear(torch.nn.Linear(200, 130))
    lin = lin.to(torch.bfloat16)
    assert lin.qweight.dtype == FP8 and lin.scales.dtype == torch.float32 and lin.bias.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        FP8Linear(torch.zeros(8, 8), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="scales"):
        FP8Linear(_fp8(130, 8), torch.zeros(1, 1))

    class Dense(torch.nn.Module):
        def __init__(self, inter):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(64, inter), torch.nn.Linear(64, inter)
            self.down_proj = torch.nn.Linear(inter, 64)

    mlp = FP8MLP.from_mlp(Dense(128))
    assert mlp.gate_up_proj.qweight.shape == (256, 64) and mlp.gate_up_proj.scales.shape == (2, 1)
    with pytest.raises(ValueError, match="whole blocks"):
        FP8MLP.from_mlp(Dense(100))
