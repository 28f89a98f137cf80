"""The int8 linear path's host checks: shapes, dtypes, devices and the C ABI's own, and the
weight quantizer, which is torch on any device (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels import fused_rmsnorm_int8, fused_swiglu_int8, quantize_int8, w8a8_gemm
from slipstream_amd.quantized import W8A8Linear, W8A8MLP, quantize_weight_int8

FAKE = 1 << 20  # a 16-byte aligned address that no refused call reads


def _gemm_args(**change):
    a = {"q": torch.zeros(2, 3, 32, dtype=torch.int8), "scale": torch.zeros(2, 3),
         "qweight": torch.zeros(8, 32, dtype=torch.int8), "w_scale": torch.zeros(8), "bias": None}
    return {**a, **change}


@pytest.mark.parametrize("change,match", [
    ({"q": torch.zeros(2, 3, 32)}, "must be int8"),
    ({"q": torch.zeros(2, 3, 32, dtype=torch.uint8)}, "must be int8"),
    ({"qweight": torch.zeros(8, 32, dtype=torch.int32)}, "must be int8"),
    ({"qweight": torch.zeros(8, 4, 8, dtype=torch.int8)}, "2-D"),
    ({"qweight": torch.zeros(8, 31, dtype=torch.int8)}, "31 input features"),
    ({"scale": torch.zeros(2, 3, dtype=torch.bfloat16)}, "float32"),
    ({"w_scale": torch.zeros(8, dtype=torch.float64)}, "float32"),
    ({"scale": torch.zeros(6)}, "one for each row"),
    ({"scale": torch.zeros(2, 3, 1)}, "one for each row"),
    ({"w_scale": torch.zeros(8, 1)}, "w_scale"),
    ({"w_scale": torch.zeros(1)}, "w_scale"),
    ({"bias": torch.zeros(1)}, "bias"),
    ({"bias": torch.zeros(9)}, "bias"),
])
def test_gemm_refuses_shapes_and_dtypes(change, match):
    with pytest.raises(ValueError, match=match):
        w8a8_gemm(**_gemm_args(**change))


def test_gemm_refuses_other_output_and_bias_types():
    with pytest.raises(_ffi.KernelError, match="not supported"):
        w8a8_gemm(**_gemm_args(), out_dtype=torch.float64)
    with pytest.raises(_ffi.KernelError, match="not supported"):
        w8a8_gemm(**_gemm_args(bias=torch.zeros(8, dtype=torch.int32)))


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="HIP devices only"):
        w8a8_gemm(**_gemm_args())
    x, w = torch.zeros(2, 32), torch.ones(32)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        quantize_int8(x)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        fused_rmsnorm_int8(x, w, x)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        fused_swiglu_int8(x, x)


def test_empty_calls_compute_nothing():
    """No tokens, no channels, no columns: the shapes come back, without a device."""
    assert w8a8_gemm(**_gemm_args(q=torch.zeros(0, 32, dtype=torch.int8), scale=torch.zeros(0))).shape == (0, 8)
    assert w8a8_gemm(**_gemm_args(qweight=torch.zeros(0, 32, dtype=torch.int8), w_scale=torch.zeros(0))).shape == (2, 3, 0)
    q, scale = quantize_int8(torch.zeros(0, 5, 32))
    assert q.shape == (0, 5, 32) and scale.shape == (0, 5)
    q, scale, s = fused_rmsnorm_int8(torch.zeros(4, 0), torch.zeros(0), torch.zeros(4, 0))
    assert q.shape == (4, 0) and s.shape == (4, 0) and torch.equal(scale, torch.zeros(4))
    q, scale = fused_swiglu_int8(torch.zeros(4, 0), torch.zeros(4, 0))
    assert torch.equal(scale, torch.zeros(4))


def test_rows_refuse_shapes_and_dtypes():
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="weight numel"):
        fused_rmsnorm_int8(x, torch.zeros(31, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="residual"):
        fused_rmsnorm_int8(x, torch.zeros(32, dtype=torch.bfloat16), x[:1])
    with pytest.raises(ValueError, match="share a dtype"):
        fused_rmsnorm_int8(x, torch.zeros(32))
    with pytest.raises(ValueError, match="share shape"):
        fused_swiglu_int8(x, x[:, :16])
    with pytest.raises(ValueError, match="share shape"):
        fused_swiglu_int8(x, x.float())
    with pytest.raises(ValueError, match="at least one dimension"):
        quantize_int8(torch.zeros(()))
    for bad in (torch.float64, torch.int8, torch.int32):
        with pytest.raises(_ffi.KernelError, match="not supported"):
            quantize_int8(torch.zeros(2, 32, dtype=bad))


def _plan(m, n, k):
    plan = (ctypes.c_int32 * 5)()
    assert _ffi.lib().ss_w8a8_plan(m, n, k, plan) == _ffi.SS_OK
    return list(plan)


def test_gpu_tests_reach_the_kernels_they_name():
    """The shapes of the product's GPU tests lie where the fitted estimates choose the kernel, tile, waves
    and split that their names say."""
    from tests.test_gpu_int8_gemm import ONCE_STREAMS, VARIANTS

    seen = set()
    for once_only, variants in ((False, VARIANTS), (True, ONCE_STREAMS)):
        for what, shapes in variants:
            name, *numbers = what.split()
            numbers = [int(v) for v in numbers]
            for shape in shapes:
                kernel, tokens, channels, parts, once = _plan(*shape)
                if name == "stream":
                    mt, nt, waves = numbers
                    assert [kernel, tokens, channels, parts] == [1, 16 * mt, 16 * nt, waves], (what, shape)
                    assert once or not once_only, (what, shape)
                else:
                    assert [kernel, tokens, channels] == [2, *numbers], (what, shape)
                    assert (parts > 1, once) == (name == "split", name == "once"), (what, shape)
            seen.add((name, *numbers))
    tiles = {(256, 256), (224, 256), (192, 256), (160, 256), (128, 256), (256, 128), (192, 128), (128, 128), (96, 128),
             (64, 128)}
    for name in ("tile", "split", "once"):
        assert {v[1:] for v in seen if v[0] == name} == tiles


def test_plan_of_calls_without_one():
    assert _plan(0, 8, 32) == _plan(4, 0, 32) == _plan(4, 8, 0) == [0] * 5
    assert _plan(1, 28672, 4095) == _plan(1, 28672, 4096)  # a copy of whole rows first
    lib, plan = _ffi.lib(), (ctypes.c_int32 * 5)()
    assert lib.ss_w8a8_plan(4, 8, 32, None) == _ffi.SS_ERR_INVALID
    assert lib.ss_w8a8_plan(-1, 8, 32, plan) == _ffi.SS_ERR_INVALID
    assert lib.ss_w8a8_plan(4, 8, 1 << 17, plan) == _ffi.SS_ERR_UNSUPPORTED
    # more results than the tile kernel's launches hold: the general kernel's refusal, or its work
    assert _plan((1 << 31) - 1, (1 << 31) - 1, 16)[0] == 0


def test_c_abi_refusals_need_no_device():
    lib = _ffi.lib()
    bf16 = _ffi.SS_DTYPE_BF16
    need = ctypes.c_int64(-1)

    def gemm(x=FAKE, xs=FAKE, w=FAKE, ws=FAKE, bias=None, out=FAKE, m=4, n=8, k=32, x_stride=32, w_stride=32,
             o_stride=8, out_dtype=bf16, bias_dtype=bf16):
        return lib.ss_w8a8_gemm(x, xs, w, ws, bias, out, m, n, k, x_stride, w_stride, o_stride, out_dtype, bias_dtype,
                                None, 0, None)

    assert gemm(m=0, x=None, out=None) == _ffi.SS_OK
    assert gemm(n=0, w=None, out=None) == _ffi.SS_OK
    for null in ("x", "xs", "w", "ws", "out"):
        assert gemm(**{null: None}) == _ffi.SS_ERR_INVALID
        assert b"null" in lib.ss_last_error()
    for neg in ("m", "n", "k"):
        assert gemm(**{neg: -1}) == _ffi.SS_ERR_INVALID
    assert gemm(x_stride=31) == _ffi.SS_ERR_INVALID
    assert gemm(w_stride=31) == _ffi.SS_ERR_INVALID
    assert gemm(o_stride=7) == _ffi.SS_ERR_INVALID
    assert gemm(out_dtype=7) == _ffi.SS_ERR_UNSUPPORTED
    assert gemm(bias=FAKE, bias_dtype=7) == _ffi.SS_ERR_UNSUPPORTED
    # 128 * 128 * 131072 = 2^31 would leave the int32 sum
    assert gemm(k=1 << 17, x_stride=1 << 17, w_stride=1 << 17) == _ffi.SS_ERR_UNSUPPORTED
    assert b"131072" in lib.ss_last_error()
    assert lib.ss_w8a8_workspace_size(4, 8, 1 << 17, 1, 1, ctypes.byref(need)) == _ffi.SS_ERR_UNSUPPORTED
    assert lib.ss_w8a8_workspace_size(-1, 8, 32, 1, 1, ctypes.byref(need)) == _ffi.SS_ERR_INVALID
    assert lib.ss_w8a8_workspace_size(4, 8, 32, 1, 1, None) == _ffi.SS_ERR_INVALID
    for k, x_whole, w_whole, copies in ((32, 1, 1, 0), (32, 0, 1, 4 * 32), (32, 1, 0, 8 * 32), (33, 1, 1, 12 * 48)):
        assert lib.ss_w8a8_workspace_size(4, 8, k, x_whole, w_whole, ctypes.byref(need)) == _ffi.SS_OK
        assert need.value == copies
    # 128 tokens of a long row, few tiles: int32 sums of several ranges
    assert lib.ss_w8a8_workspace_size(197, 4096, 14336, 1, 1, ctypes.byref(need)) == _ffi.SS_OK
    ranges, rest = divmod(need.value, 197 * 4096 * 4)
    assert ranges > 1 and rest == 0

    def rows(x=FAKE, q=FAKE, scale=FAKE, m=4, k=32, stride=32, dtype=bf16):
        return (lib.ss_quantize_int8(x, q, scale, m, k, stride, dtype, None),
                lib.ss_rmsnorm_int8(x, FAKE, FAKE, q, scale, FAKE, m, k, stride, 32, 1e-6, dtype, None),
                lib.ss_swiglu_int8(x, FAKE, q, scale, m, k, stride, 32, dtype, None))

    assert set(rows(m=0, x=None)) == set(rows(k=0, x=None)) == {_ffi.SS_OK}
    for bad in ({"x": None}, {"q": None}, {"scale": None}, {"m": -1}, {"k": -1}, {"stride": -32}):
        assert set(rows(**bad)) == {_ffi.SS_ERR_INVALID}, bad
    for bad in ({"dtype": 9}, {"m": 1 << 31}, {"k": 1 << 29}):
        assert set(rows(**bad)) == {_ffi.SS_ERR_UNSUPPORTED}, bad
    # a residual needs somewhere for the sum
    assert lib.ss_rmsnorm_int8(FAKE, FAKE, FAKE, FAKE, FAKE, None, 4, 32, 32, 32, 1e-6, bf16, None) == _ffi.SS_ERR_INVALID


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weight_quantizer(dtype):
    """Within half a step of the weight (and the roundings of 127 / max and the product,
    2^-24 of 127 each), the largest at 127; a channel of zeros has scale 0."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(37, 251, generator=g).to(dtype)
    w[5] = 0
    q, scale = quantize_weight_int8(w)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == (37,)
    top = w.double().abs().amax(1)
    assert torch.equal(q[5], torch.zeros_like(q[5])) and scale[5] == 0
    live = top > 0
    assert (scale[live].double() / (top[live] / 127) - 1).abs().max() <= 2.0**-24
    steps = w[live].double() * 127 / top[live, None]
    assert (q[live].double() - steps).abs().max() <= 0.5 + 127 * 2 * 2.0**-24
    assert torch.equal(q[live].abs().amax(1), torch.full((36,), 127, dtype=torch.int8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weight_quantizer_rounds_twice(dtype):
    """Bit for bit ``127 / max`` rounded to fp32, its product with the weight rounded to fp32, and that to
    an integer: both roundings here by doubles, which hold a product of two fp32 values and round
    a quotient of two so that rounding it again to fp32 is the quotient's nearest."""
    w = torch.randn(67, 1021, generator=torch.Generator().manual_seed(2)).to(dtype)
    q, scale = quantize_weight_int8(w)
    top = w.double().abs().amax(1, keepdim=True)
    steps = (w.double() * (127 / top).float().double()).float()
    assert torch.equal(q, torch.round(steps).to(torch.int8))
    assert torch.equal(scale, (top / 127).float()[:, 0])


def test_weight_quantizer_and_modules_refuse():
    with pytest.raises(ValueError, match="2-D"):
        quantize_weight_int8(torch.zeros(4))
    for bad in (float("inf"), float("nan")):
        with pytest.raises(ValueError, match="infinities or NaN"):
            quantize_weight_int8(torch.tensor([[1.0, bad]]))
    q, s = quantize_weight_int8(torch.randn(6, 4))
    with pytest.raises(ValueError, match="int8"):
        W8A8Linear(q.float(), s)
    with pytest.raises(ValueError, match="float32"):
        W8A8Linear(q, s[:5])
    with pytest.raises(ValueError, match="float32"):
        W8A8Linear(q, s.half())
    lin = W8A8Linear(q, s)
    with pytest.raises(ValueError, match="share in/out"):
        W8A8MLP(lin, W8A8Linear(q[:5], s[:5]), lin)
    with pytest.raises(ValueError, match="down_proj reads"):
        W8A8MLP(lin, lin, lin)


def test_mlp_stacks_gate_and_up():
    """The stacked projection's rows are the two weights' own, and its bias theirs, with zeros
    for one that has none."""
    torch.manual_seed(0)
    mlp = torch.nn.Module()
    mlp.gate_proj = torch.nn.Linear(16, 24, bias=True)
    mlp.up_proj = torch.nn.Linear(16, 24, bias=False)
    mlp.down_proj = torch.nn.Linear(24, 16, bias=True)
    m = W8A8MLP.from_mlp(mlp)
    for part, lin in ((slice(0, 24), mlp.gate_proj), (slice(24, 48), mlp.up_proj)):
        q, s = quantize_weight_int8(lin.weight.detach())
        assert torch.equal(m.gate_up_proj.qweight[part], q) and torch.equal(m.gate_up_proj.scales[part], s)
    assert torch.equal(m.gate_up_proj.bias, torch.cat([mlp.gate_proj.bias, torch.zeros(24)]))
    assert torch.equal(m.down_proj.bias, mlp.down_proj.bias)
