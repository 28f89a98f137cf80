"""e4m3 rows and the block-scaled product on the GPU, against the float64 oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ora
from slipstream_amd import _ffi
from slipstream_amd.kernels import fp8_gemm, quantize_fp8
from slipstream_amd.kernels.fp8_rows import FP8
from slipstream_amd.quantized import FP8MLP, FP8Linear

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _f64(t):
    return t.detach().cpu().double().numpy()


def _check_rows(x, q, scale):
    want_q, want_scale = ora.quantize_rows(_f64(x).reshape(-1, x.shape[-1]))
    assert np.array_equal(_f64(q).reshape(want_q.shape), want_q)
    assert np.array_equal(_f64(scale).reshape(want_scale.shape), want_scale.astype(np.float64), equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (17, 129), (16, 256), (33, 2051), (5, 4096), (197, 640)])
def test_rows_are_exact(device, dtype, m, k):
    gen = torch.Generator().manual_seed(m * 7919 + k)
    x = (torch.randn(m, k, generator=gen) * torch.exp(2 * torch.randn(m, 1, generator=gen))).to(dtype)
    q, scale = quantize_fp8(x.cuda())
    assert q.dtype == FP8 and q.shape == x.shape and scale.dtype == torch.float32
    assert scale.shape == (m, -(-k // 128)) and (m == 1 or scale.stride(0) == 1)
    _check_rows(x, q, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_halfway_quotients_go_to_the_even_value(device, dtype):
    """Largest magnitudes of 448 times a power of two: quotients are the values themselves, all halfway
    points of e4m3 among them; and 7/8 of that, where the rounded reciprocal is off."""
    codes = torch.arange(256, dtype=torch.uint8).view(FP8).double()
    values = codes[codes.isfinite()].unique()
    points = torch.cat([values, (values[1:] + values[:-1]) / 2])
    rows = []
    for top in (448.0, 392.0, 7.0, 3.5 * 2.0**-7):
        p = (points * (top / 448.0)).to(dtype)
        p = p[p.double().abs() <= top]
        for part in p.split(127):
            part = torch.nn.functional.pad(part, (0, 127 - part.numel()))
            rows.append(torch.cat([torch.tensor([top], dtype=dtype), part]))
    x = torch.stack(rows)
    _check_rows(x, *quantize_fp8(x.cuda()))


def test_fp32_quotients_next_to_a_halfway_point(device):
    """Neighbours in fp32 of halfway points, for largest magnitudes with all their bits in use."""
    gen = torch.Generator().manual_seed(5)
    values = torch.arange(256, dtype=torch.uint8).view(FP8).double()
    values = values[values.isfinite()].unique()
    half = (values[1:] + values[:-1]) / 2
    rows = []
    for top in (448.0 * torch.rand(40, generator=gen) + 1).tolist():
        top = float(np.float32(top))
        at = (half[torch.randint(0, len(half), (42,), generator=gen)] * top / 448.0).float()
        inf = torch.tensor(float("inf"))
        row = torch.cat([at, torch.nextafter(at, inf), torch.nextafter(at, -inf)]).clamp(-top, top)
        rows.append(torch.cat([torch.tensor([top, 0.0]), row]))
    x = torch.stack(rows)
    _check_rows(x, *quantize_fp8(x.cuda()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_extreme_blocks(device, dtype):
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    x = torch.zeros(8, 300, dtype=dtype)
    x[0, 5], x[0, 130], x[0, 299] = big, -big, tiny  # a block each; the last one is short
    x[1, 0], x[1, 1] = float("inf"), 1.0
    x[2, 128], x[2, 3] = float("nan"), 2.0
    x[3, :] = tiny
    x[4, 10] = torch.finfo(dtype).smallest_normal / 4  # subnormal
    x[5, 256:] = -3.0
    x[6, 7], x[6, 200] = -float("inf"), 5.0
    q, scale = quantize_fp8(x.cuda())
    _check_rows(x, q, scale)
    assert scale[1, 0].isnan() and not q[1, :128].float().any() and scale[2, 0].isfinite() and scale[2, 1].isnan()


def test_rows_of_any_layout(device):
    gen = torch.Generator().manual_seed(11)
    base = torch.randn(2, 9, 515, generator=gen).to(torch.bfloat16)
    for x in (base[:, :, 1:402], base[:, ::2, 3:], base.transpose(0, 1), base[..., ::2], base[1, :, 5:6]):
        q, scale = quantize_fp8(x.cuda() if x.is_contiguous() else _same_layout(x))
        _check_rows(x, q, scale)


def _same_layout(x):
    base = torch.zeros(x.untyped_storage().nbytes() // x.element_size(), dtype=x.dtype, device="cuda")
    out = base.as_strided(x.shape, x.stride(), x.storage_offset())
    out.copy_(x)
    return out


# ---- the product ---------------------------------------------------------------------------


def _operands(m, n, k, seed, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))
    w = torch.randn(n, k, generator=gen) * k**-0.5
    kb = -(-k // 128)
    q = (torch.randn(m, k, generator=gen) * 100).clamp(-448, 448).to(FP8)
    qw = (torch.randn(n, k, generator=gen) * 100).clamp(-448, 448).to(FP8)
    scale = torch.rand(m, kb, generator=gen) * 0.01 + 0.001
    ws = (torch.rand(-(-n // 128), kb, generator=gen) + 0.1) * 0.01
    return [t.to(device) for t in (q, scale, qw, ws)]


def _check_gemm(out, q, scale, qw, ws, bias=None):
    """To fp16 and fp32 a block's 128 products are exact in fp32 and their sum has at most 127 roundings of the
    partial sums, each below 2^-23 of the terms' magnitudes (to the nearest or truncated); the scales' product
    and the sum over blocks add two and one more a block, the bias one; and half a step of the output's type.
    To bf16 the e4m3 instruction sums a block, by its measured bound 2^-15.4 of the magnitudes: the 2^-15.98
    here stands for that beside the half step, which is 2^-8."""
    want, size = ora.gemm(_f64(q).reshape(-1, q.shape[-1]), _f64(scale).reshape(-1, scale.shape[-1]), _f64(qw),
                          _f64(ws), None if bias is None else _f64(bias))
    got = _f64(out).reshape(want.shape)
    tol = HALF_STEP[out.dtype] * np.abs(want) + 2.0**-23 * (130 + scale.shape[-1]) * size
    err = np.abs(got - want)
    assert np.isfinite(got).all() and (err <= tol).all(), (err - tol).max()


SHAPES = [(1, 1, 1), (1, 130, 128), (3, 64, 127), (5, 300, 129), (8, 128, 512), (16, 4096, 896), (17, 257, 2051),
          (33, 1152, 896), (64, 512, 1024), (65, 640, 4096), (100, 4999, 256), (128, 256, 144), (197, 1000, 2048),
          (256, 384, 1408), (300, 2000, 272), (513, 640, 1024)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gemm(device, m, n, k, dtype):
    q, scale, qw, ws = _operands(m, n, k, m + 31 * n + 1009 * k)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).cuda() if (m + n) % 2 else None
    _check_gemm(fp8_gemm(q, scale, qw, ws, bias, dtype), q, scale, qw, ws, bias)


@pytest.mark.parametrize("m", [1, 24, 300])
def test_gemm_layouts(device, m):
    """Scales block by block or row by row, rows apart, unaligned rows, three dimensions, bias of any type."""
    n, k = 384, 640
    q, scale, qw, ws = _operands(m, n, k, m)
    want = fp8_gemm(q, scale, qw, ws, None, torch.float32)
    _check_gemm(want, q, scale, qw, ws)
    assert torch.equal(fp8_gemm(q, scale.t().contiguous().t(), qw, ws, None, torch.float32), want)
    wide = torch.zeros(m, k + 48, dtype=torch.uint8, device="cuda").view(FP8)
    wide.view(torch.uint8)[:, 16 : 16 + k] = q.view(torch.uint8)
    assert torch.equal(fp8_gemm(wide[:, 16 : 16 + k], scale, qw, ws, None, torch.float32), want)
    odd = torch.zeros(n * (k + 3) + 1, dtype=torch.uint8, device="cuda").view(FP8)[1:].view(n, k + 3)
    odd.view(torch.uint8)[:, :k] = qw.view(torch.uint8)
    _check_gemm(fp8_gemm(q, scale, odd[:, :k], ws, None, torch.float32), q, scale, qw, ws)
    big = torch.zeros(3, 10, device="cuda")
    big[:, 2 : 2 + ws.shape[1]] = ws
    assert torch.equal(fp8_gemm(q, scale, qw, big[:, 2 : 2 + ws.shape[1]], None, torch.float32), want)
    if m % 3 == 0:
        q3, s3 = q.view(3, m // 3, k), scale.view(3, m // 3, -1)
        out = fp8_gemm(q3, s3, qw, ws, None, torch.float32)
        assert out.shape == (3, m // 3, n) and torch.equal(out.view(m, n), want)
        s3 = scale.t().contiguous().view(-1, 3, m // 3).movedim(0, -1)  # as quantize_fp8 leaves it
        assert torch.equal(fp8_gemm(q3, s3, qw, ws, None, torch.float32).view(m, n), want)
    for bias_type in (torch.float16, torch.bfloat16, torch.float32):
        bias = torch.randn(n, device="cuda").to(bias_type)
        _check_gemm(fp8_gemm(q, scale, qw, ws, bias, torch.bfloat16), q, scale, qw, ws, bias)


def test_gemm_without_columns_is_the_bias(device):
    q = torch.zeros(5, 0, dtype=torch.uint8, device="cuda").view(FP8)
    qw = torch.zeros(130, 0, dtype=torch.uint8, device="cuda").view(FP8)
    bias = torch.randn(130, device="cuda")
    out = fp8_gemm(q, torch.zeros(5, 0, device="cuda"), qw, torch.zeros(2, 0, device="cuda"), bias, torch.float32)
    assert torch.equal(out, bias.expand(5, 130))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_bad_block_stays_in_its_row(device, m):
    """A NaN scale (a block that held a NaN) makes its row NaN and no other."""
    q, scale, qw, ws = _operands(m, 256, 384, 3)
    scale[m // 2, 1] = float("nan")
    out = fp8_gemm(q, scale, qw, ws)
    bad = out.isnan().all(dim=1)
    assert bad[m // 2] and bad.sum() == 1 and out.isnan().sum() == 256


@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (24, 1152, 896), (64, 640, 2048), (300, 384, 4096)])
def test_gemm_repeats_itself_and_without_a_workspace_is_right(device, m, n, k):
    q, scale, qw, ws = _operands(m, n, k, 99)
    first = fp8_gemm(q, scale, qw, ws)
    for _ in range(3):
        assert torch.equal(fp8_gemm(q, scale, qw, ws), first)
    out = torch.empty(m, n, dtype=torch.float32, device="cuda")
    status = _ffi.lib().ss_fp8_gemm(q.data_ptr(), scale.data_ptr(), qw.data_ptr(), ws.data_ptr(), None, out.data_ptr(), m,
                                    n, k, k, k, n, _ffi.i64x2(*scale.stride()), _ffi.i64x2(*ws.stride()),
                                    _ffi.SS_DTYPE_F32, 0, None, 0, _ffi.stream_ptr(q.device))
    _ffi.check(status, "fp8_gemm")
    _check_gemm(out, q, scale, qw, ws)


def test_linear_and_mlp_together(device):
    """Rows quantized, gate and up, SwiGLU, rows, down: as the layer runs them, and captured in a graph
    that is replayed with new inputs between eager calls."""
    torch.manual_seed(2)

    class Dense(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(256, 384, bias=False), torch.nn.Linear(256, 384)
            self.down_proj = torch.nn.Linear(384, 256)

    mlp = FP8MLP.from_mlp(Dense()).cuda().to(torch.bfloat16)
    lin = FP8Linear.from_linear(torch.nn.Linear(256, 200)).cuda().to(torch.bfloat16)
    x = torch.randn(3, 7, 256, device="cuda").to(torch.bfloat16)
    q, scale = quantize_fp8(x)
    out = lin(x)
    assert out.shape == (3, 7, 200)
    _check_gemm(out, q, scale, lin.qweight, lin.scales, lin.bias)
    assert torch.equal(mlp(x), mlp.forward_fp8(q, scale, x.dtype))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin(x), mlp(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = lin(x), mlp(x)
    for seed in range(3):
        x.copy_(torch.randn(3, 7, 256, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lin(x)) and torch.equal(z, mlp(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(2048, 8192, 640), (1000, 16384 + 200, 384), (768, 4096, 2048 + 48), (500, 1280, 4096)])
def test_gemm_of_many_tokens(device, m, n, k, dtype):
    """The widest tiles, whole ones and cut ones, and keys split over workgroups."""
    q, scale, qw, ws = _operands(m, n, k, m + n + k)
    _check_gemm(fp8_gemm(q, scale, qw, ws, None, dtype), q, scale, qw, ws)


@pytest.mark.parametrize("n,k", [(1152, 896), (4096 + 16, 2176), (700, 5120)])
@pytest.mark.parametrize("m", [1, 2, 8, 9, 16, 17, 32, 33, 48, 65, 96, 128])
def test_gemm_of_few_tokens(device, m, n, k):
    """The stream kernel's tiles, its waves' shares of the keys and rows that end inside a tile."""
    q, scale, qw, ws = _operands(m, n, k, 7 * m + n)
    for dtype in (torch.bfloat16, torch.float16):
        _check_gemm(fp8_gemm(q, scale, qw, ws, None, dtype), q, scale, qw, ws)


def test_gemm_of_very_long_rows(device):
    """Rows longer than the DMA kernels' descriptors reach over a tile of them."""
    q, scale, qw, ws = _operands(3, 130, (1 << 21) + 144, 17)
    for rows in (q, q[:1]):
        _check_gemm(fp8_gemm(rows, scale[: len(rows)], qw, ws, None, torch.float32), rows, scale[: len(rows)], qw, ws)
