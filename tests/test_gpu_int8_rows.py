"""Rows quantized to int8 (plain, behind the RMS norm with the residual, behind SwiGLU) against
the formulas in 64 bits.

Tolerances, in units of u = 2^-24 (a fp32 rounding, relative):
  q: the value in steps is y * 127 / a; 1 / a, its product with 127 and the product with y are
     rounded once each, the norm's s * w once in y and once in a (exact for 16-bit types), so
     |q - steps| <= 1/2 + 127 * 5 u. SwiGLU: exp is within 2 u, 1 + exp and the quotient round
     once each, then * u: within 7 u in y and the same in a.
  scale: a / 127 once (a as above); the norm's sum of squares adds each of a thread's
     cols / 256 values and 16 partial sums with a rounding each, halved by the root, and the
     mean, eps, root, reciprocal and two products round once each.
"""

from __future__ import annotations

import pytest
import torch

from slipstream_amd.kernels import fused_rmsnorm, fused_rmsnorm_int8, fused_swiglu_int8, quantize_int8

pytestmark = pytest.mark.gpu

U = 2.0**-24
SMALLEST = 127 * 2.0**-126
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# one element, one piece and either side of it, odd, each count of pieces a thread, the two-pass rows
COLS = [1, 7, 8, 9, 64, 513, 896, 1000, 2051, 4096, 4864, 8192, 14336, 16384, 16392, 40001]


def _rand(g, shape, dtype, device, spread=True):
    x = torch.randn(shape, generator=g, device=device)
    if spread and len(shape) > 1:
        x = x * torch.exp(torch.randn((*shape[:-1], 1), generator=g, device=device))
    return x.to(dtype)


def _check(q, scale, y, y_err, scale_err, what):
    """int8 rows against fp64 rows ``y`` known to a relative ``y_err``."""
    assert q.dtype == torch.int8 and scale.dtype == torch.float32
    assert q.shape == y.shape and scale.shape == y.shape[:-1]
    top = y.abs().amax(-1)
    live = top >= SMALLEST
    assert not q[~live].any() and not scale[~live].any(), f"{what}: a row of zeros"
    steps = y * (127 / torch.where(live, top, 1.0))[..., None]
    off = ((q.double() - steps).abs()[live]).max().item() if live.any() else 0.0
    assert off <= 0.5 + 127 * (2 * y_err + 3 * U), f"{what}: {off} steps off"
    rel = ((scale.double() * 127 / top - 1).abs()[live]).max().item() if live.any() else 0.0
    assert rel <= scale_err, f"{what}: scale {rel / U:.1f} u off"
    assert (q[live].abs().amax(-1) == 127).all()


def _norm64(x, w, r, eps):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    s64 = s.double()
    return s64 * w.double() / (s64.square().mean(-1, keepdim=True) + eps).sqrt(), s


def _norm_scale_err(cols):
    return ((cols / 256 + 16 + 16) / 2 + 10) * U


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_rows(device, dtype, cols):
    g = torch.Generator(device=device).manual_seed(cols)
    x = _rand(g, (5, cols), dtype, device)
    x[3] = 0
    q, scale = quantize_int8(x)
    _check(q, scale, x.double(), 0.0, 2 * U, f"rows {cols} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_are_what_elementary_operations_give(device, dtype):
    """Bit for bit: the reciprocal of the row's maximum, its product with 127 and the product with
    the value, rounded to fp32 each."""
    g = torch.Generator(device=device).manual_seed(17)
    x = _rand(g, (333, 2051), dtype, device)
    top = x.float().abs().amax(-1, keepdim=True)
    q, scale = quantize_int8(x)
    assert torch.equal(q, torch.round(x.float() * (127 * torch.reciprocal(top))).to(torch.int8))
    assert torch.equal(scale, (top.double() / 127).float()[:, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_is_quantized_as_its_rows_are(device, dtype):
    """Values far on either side of zero, the divisor's overflow included, in rows of their own."""
    at = torch.tensor([-1e4, -103.0, -89.0, -88.5, -70.0, -69.0, -20.0, -1.0, 0.0, 1.0, 20.0, 90.0, 1e4], device=device)
    gate = at.to(dtype)[:, None].expand(-1, 40).contiguous()
    up = torch.linspace(-1, 1, 40, device=device).to(dtype).expand(13, -1)
    q, scale = fused_swiglu_int8(gate, up)
    assert torch.isfinite(scale).all()
    g64 = gate.double()
    y = g64 / (1 + torch.exp(-g64)) * up.double()
    normal = (at.to(dtype).float() > -80) & (at != 0)  # below, up to 2^-100 is dropped
    _check(q[normal], scale[normal], y[normal], 7 * U, 9 * U, f"far {dtype}")
    rest = (q.double() * scale.double()[:, None] - y)[~normal]
    assert rest.abs().max().item() <= 2.0**-100


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(device, dtype, cols, with_residual):
    g = torch.Generator(device=device).manual_seed(cols)
    x = _rand(g, (2, 2, cols), dtype, device)
    w = (1 + 0.1 * _rand(g, (cols,), torch.float32, device)).to(dtype)
    r = _rand(g, (2, 2, cols), dtype, device) if with_residual else None
    x[1, 0] = 0
    if with_residual:
        r[1, 0] = 0
    q, scale, s = fused_rmsnorm_int8(x, w, r, 1e-6)
    y, want = _norm64(x, w, r, 1e-6)
    if with_residual:
        assert s.dtype == dtype and torch.equal(s, want) and s.data_ptr() not in (x.data_ptr(), r.data_ptr())
    else:
        assert s is None
    _check(q, scale, y, U if dtype == torch.float32 else 0.0, _norm_scale_err(cols), f"norm {cols} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_swiglu(device, dtype, cols):
    g = torch.Generator(device=device).manual_seed(cols)
    gate, up = 2 * _rand(g, (5, cols), dtype, device), _rand(g, (5, cols), dtype, device)
    up[2] = 0
    q, scale = fused_swiglu_int8(gate, up)
    g64 = gate.double()
    err = 7 * U
    _check(q, scale, g64 / (1 + torch.exp(-g64)) * up.double(), err, err + 2 * U, f"swiglu {cols} {dtype}")


@pytest.mark.parametrize("rows", [1, 3, 257, 2240])
def test_row_counts_agree(device, rows):
    """A row's int8 values and scale do not depend on the rows around it."""
    g = torch.Generator(device=device).manual_seed(rows)
    x, r = (_rand(g, (rows, 1024), torch.bfloat16, device) for _ in range(2))
    w = torch.ones(1024, device=device, dtype=torch.bfloat16)
    q, scale, s = fused_rmsnorm_int8(x, w, r)
    at = rows // 2
    q1, scale1, s1 = fused_rmsnorm_int8(x[at], w, r[at])
    assert scale1.shape == () and torch.equal(q[at], q1) and torch.equal(scale[at], scale1) and torch.equal(s[at], s1)
    y, _ = _norm64(x, w, r, 1e-6)
    _check(q, scale, y, 0.0, _norm_scale_err(1024), f"{rows} rows")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 4096, 40001])
def test_norm_rounds_exact_halves_to_even(device, dtype, cols):
    """Normalised rows of few bits hold many exact halves of a step, and q is the nearest integer of
    the exact quotient, found here in whole numbers: with p = x * w and a = max |p|,
    |q| = floor((254 |p| + a) / 2 a), less one where that was a half and gives an odd number."""
    g = torch.Generator(device="cpu").manual_seed(cols)
    x = torch.randint(-254, 255, (33, cols), generator=g)
    w = torch.randint(1, 4, (cols,), generator=g)
    q, scale, _ = fused_rmsnorm_int8(x.to(device, dtype), w.to(device, dtype))
    p = x * w
    top = p.abs().amax(-1, keepdim=True)
    num = 254 * p.abs() + top
    n = num // (2 * top)
    half = (num % (2 * top) == 0) & (top > 0)
    n = torch.where(half & (n % 2 == 1), n - 1, n)
    assert half.sum().item() > 0
    assert torch.equal(q.cpu().long(), n * p.sign())


def test_norm_in_int8_is_the_norm(device):
    """The int8 rows stand for what ``fused_rmsnorm`` gives: within half a step and that
    op's two roundings to bf16 (2^-8 of the value each)."""
    g = torch.Generator(device=device).manual_seed(5)
    x, r = (_rand(g, (17, 4096), torch.bfloat16, device) for _ in range(2))
    w = (1 + 0.1 * torch.randn(4096, generator=g, device=device)).to(torch.bfloat16)
    q, scale, _ = fused_rmsnorm_int8(x, w, r)
    y = fused_rmsnorm(x, w, r).double()
    off = (q.double() * scale.double()[:, None] - y).abs()
    assert (off <= 0.501 * scale.double()[:, None] + 2 * 2.0**-8 * y.abs() * 1.01).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 1001, 4096, 40001])
def test_nan_and_infinity_mark_their_row_only(device, dtype, cols):
    g = torch.Generator(device=device).manual_seed(cols)
    x = _rand(g, (6, cols), dtype, device)
    good = x.clone()
    for row, v in ((0, float("nan")), (2, float("inf")), (5, float("-inf"))):
        x[row, (cols * 3) // 4] = v
    w, one = torch.ones(cols, device=device, dtype=dtype), torch.ones_like(x)
    zero = torch.zeros_like(x)
    for what, call in (("rows", lambda t: quantize_int8(t)), ("norm", lambda t: fused_rmsnorm_int8(t, w)[:2]),
                       ("residual", lambda t: fused_rmsnorm_int8(zero, w, t)[:2]),
                       ("up", lambda t: fused_swiglu_int8(one, t))):
        q, scale = call(x)
        q0, scale0 = call(good)
        for row in range(6):
            if row in (0, 2, 5):
                assert torch.isnan(scale[row]) and not q[row].any(), what
            else:
                assert torch.equal(q[row], q0[row]) and torch.equal(scale[row], scale0[row]), what
    _, scale = fused_swiglu_int8(x, one)
    assert torch.isnan(scale[[0, 2, 5]]).all() and torch.isfinite(scale[[1, 3, 4]]).all()


def test_smallest_and_largest_rows(device):
    """Either side of the smallest scale, subnormal rows, and rows next to the largest number."""
    big = torch.finfo(torch.float32).max
    tops = [1e-45, 1e-38, SMALLEST * 0.999, SMALLEST, SMALLEST * 1.01, 1e-30, 1.0, big / 3, big]
    base = torch.tensor([1.0, -0.5, 0.25, 0.0, -1.0 / 127, 3.0 / 127], device=device)
    x = torch.stack([base * t for t in tops])
    q, scale = quantize_int8(x)
    assert torch.isfinite(scale).all()
    _check(q, scale, x.double(), 0.0, 2 * U, "extremes")
    assert q[-1].tolist()[:2] == [127, -64]  # 63.5 rounds to even


def test_ties_round_to_even(device):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5, 126.5]], device=device)
    q, scale = quantize_int8(x)
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 64, 126]] and scale.item() == 1.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignments(device, dtype):
    """Rows of wider buffers, at every element offset, transposed and broadcast ones: as the
    contiguous rows give, and nothing else is read into them."""
    g = torch.Generator(device=device).manual_seed(3)
    buf = torch.full((7, 2 * 1000 + 24), 1e4, device=device, dtype=dtype)
    for off in (0, 1, 3, 8):
        gate, up = buf[:, off : off + 1000], buf[:, off + 1008 : off + 2008]
        gate.copy_(torch.randn(gate.shape, generator=g, device=device))
        up.copy_(torch.randn(up.shape, generator=g, device=device))
        w = buf[0, off : off + 1000]
        cg, cu, cw = gate.clone(), up.clone(), w.clone()
        for got, want in ((quantize_int8(up), quantize_int8(cu)), (fused_swiglu_int8(gate, up), fused_swiglu_int8(cg, cu)),
                          (fused_rmsnorm_int8(gate, w, up), fused_rmsnorm_int8(cg, cw, cu))):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), off
        _check(*quantize_int8(up), cu.double(), 0.0, 2 * U, f"offset {off}")
        buf.fill_(1e4)
    t = torch.randn(64, 9, generator=g, device=device).to(dtype).t()
    assert all(torch.equal(a, b) for a, b in zip(quantize_int8(t), quantize_int8(t.contiguous())))
    b = t[:1].expand(4, 64)
    q, scale = quantize_int8(b)
    assert (q == q[0]).all() and (scale == scale[0]).all()


def test_nothing_is_written_past_the_rows(device):
    """The C entry's outputs in the middle of larger buffers, at an odd width."""
    from slipstream_amd import _ffi

    rows, cols = 3, 1003
    x = torch.randn(rows, cols, device=device)
    for dtype in DTYPES:
        xt = x.to(dtype)
        q = torch.full((rows * cols + 64,), 77, dtype=torch.int8, device=device)
        scale = torch.full((rows + 8,), 77.0, device=device)
        s = torch.full((rows * cols + 64,), 77.0, dtype=dtype, device=device)
        w = torch.ones(cols, dtype=dtype, device=device)
        _ffi.check(_ffi.lib().ss_rmsnorm_int8(xt.data_ptr(), xt.data_ptr(), w.data_ptr(), q[32:].data_ptr(),
                                              scale[4:].data_ptr(), s[32:].data_ptr(), rows, cols, cols, cols, 1e-6,
                                              _ffi.dtype_code(dtype), _ffi.stream_ptr(device)), "norm")
        want = fused_rmsnorm_int8(xt, w, xt)
        torch.cuda.synchronize()
        for got, ref, edge in ((q, want[0], 32), (scale, want[1], 4), (s, want[2], 32)):
            n = ref.numel()
            assert torch.equal(got[edge : edge + n], ref.reshape(-1))
            assert (got[:edge] == 77).all() and (got[edge + n :] == 77).all()


@pytest.mark.parametrize("cols", [64, 1003, 4096, 40001])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_sum_in_place(device, cols, into):
    """The C entry with the sum written over one of its addends."""
    from slipstream_amd import _ffi

    g = torch.Generator(device=device).manual_seed(cols)
    x, r = (_rand(g, (5, cols), torch.bfloat16, device) for _ in range(2))
    w = torch.ones(cols, device=device, dtype=torch.bfloat16)
    want = fused_rmsnorm_int8(x, w, r)
    q = torch.empty((5, cols), dtype=torch.int8, device=device)
    scale = torch.empty(5, device=device)
    s = r if into == "residual" else x
    _ffi.check(_ffi.lib().ss_rmsnorm_int8(x.data_ptr(), r.data_ptr(), w.data_ptr(), q.data_ptr(), scale.data_ptr(),
                                          s.data_ptr(), 5, cols, cols, cols, 1e-6, _ffi.dtype_code(x.dtype),
                                          _ffi.stream_ptr(device)), "norm")
    assert torch.equal(q, want[0]) and torch.equal(scale, want[1]) and torch.equal(s, want[2])


def test_more_bytes_than_31_bits_hold(device):
    """Rows whose addresses pass 2^31 and 2^32 bytes: the last ones are as they are alone."""
    rows, cols = 280_000, 8192  # 4.6 GB in bf16
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=device)
    tail = torch.randn(3, cols, device=device).to(torch.bfloat16)
    x[-3:] = tail
    q, scale = quantize_int8(x)
    q1, scale1 = quantize_int8(tail)
    assert torch.equal(q[-3:], q1) and torch.equal(scale[-3:], scale1)
    assert not scale[:-3].any() and not q[rows // 2].any()


def test_more_rows_than_a_launch_holds(device):
    """17 million rows: a launch's threads stay below 2^32, so they take more than one."""
    rows, cols = 17_000_003, 8
    x = torch.arange(rows, device=device, dtype=torch.float32)[:, None].expand(rows, cols).contiguous()
    x[:, 0] += 1
    q, scale = quantize_int8(x.to(torch.bfloat16))
    assert torch.equal(scale, x.to(torch.bfloat16).float().amax(1) / torch.full((), 127.0, device=device))
    assert (q.amax(1) == 127).all()
    s, one = torch.zeros_like(x), torch.ones(cols, device=device)
    q, scale, s = fused_rmsnorm_int8(x, one, s)
    assert torch.equal(s, x) and (q.amax(1) == 127).all() and torch.isfinite(scale).all()


@pytest.mark.parametrize("rows,cols,with_residual", [(2240, 4096, True), (300, 4096, False), (300, 1003, True)])
def test_norm_differs_from_elementary_operations_at_halves_only(device, rows, cols, with_residual):
    """Rows in bf16 in which a few channels are large: the call repeats itself bit for bit, its sum is
    the elementary one, and where its q is not that of ``s * rsqrt(mean(s^2) + eps) * w`` in fp32, the
    exact quotient s w 127 / max|s w| is a half of a step, which that chain's last bits send either
    way and the kernel sends to even. s and w have 8 bits each, so doubles hold s w, 254 s w and the
    remainder exactly."""
    g = torch.Generator(device=device).manual_seed(rows + cols)

    def states():
        x = torch.randn(rows, cols, generator=g, device=device) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=device))
        return (x * torch.where(torch.rand(cols, generator=g, device=device) < 0.004, 12.0, 1.0)).to(torch.bfloat16)

    x, r = states(), states() if with_residual else None
    w = (1 + 0.1 * torch.randn(cols, generator=g, device=device)).to(torch.bfloat16)
    first = fused_rmsnorm_int8(x, w, r)
    for _ in range(3):
        assert all(a is b or torch.equal(a, b) for a, b in zip(first, fused_rmsnorm_int8(x, w, r)))
    q, scale, s = first
    hidden = x if r is None else (x.float() + r.float()).to(torch.bfloat16)
    assert s is None or torch.equal(s, hidden)
    y = hidden.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    plain = torch.round(y * (127 / y.abs().amax(-1, keepdim=True)))
    row, col = (q.float() != plain).nonzero(as_tuple=True)
    p = hidden.double() * w.double()
    top, p = p.abs().amax(-1)[row], p[row, col].abs()
    assert (torch.remainder(254 * p + top, 2 * top) == 0).all()
    assert (q[row, col] % 2 == 0).all() and (q[row, col].float() - plain[row, col]).abs().eq(1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 1003, 4096, 40001])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norm_of_zeros_and_of_rows_whose_squares_leave_fp32(device, dtype, cols, with_residual, eps):
    """A row of zeros has scale 0 whatever eps is, and rows whose squares' sum is above or below what
    fp32 holds have the norm's value as any other: the sum is taken again of the row times a power
    of two, which rounds as it does elsewhere, and the rest in doubles."""
    g = torch.Generator(device=device).manual_seed(cols)
    sizes = torch.tensor([1.0, 0.0, 2.0**60, 2.0**64, 2.0**70, 2.0**122, 2.0**-40, 2.0**-46, 2.0**-60, 2.0**-70, 2.0**-100, 0.0],
                         dtype=torch.float64, device=device)
    if dtype == torch.float16:  # from its smallest to its largest
        sizes = torch.tensor([1.0, 0.0, 2.0**12, 2.0**-10, 2.0**-24, 0.0], dtype=torch.float64, device=device)
    x = torch.randn(len(sizes), cols, generator=g, device=device).clamp(-7, 7).double()
    x = (x * sizes[:, None]).to(dtype)
    w = (1 + 0.1 * _rand(g, (cols,), torch.float32, device)).to(dtype)
    r = (x * 0.25).flip(-1) if with_residual else None
    q, scale, s = fused_rmsnorm_int8(x, w, r, eps)
    y, want = _norm64(x, w, r, eps)
    assert s is None or torch.equal(s, want)
    assert torch.isfinite(scale).all()
    p = want.double() * w.double()
    if with_residual and dtype == torch.float16:  # the sum of the smallest may be zero everywhere
        y = torch.where(p.abs().amax(-1, keepdim=True) > 0, y, 0.0)
    _check(q, scale, y, U if dtype == torch.float32 else 0.0, _norm_scale_err(cols), f"norm {cols} {dtype} {eps}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [16, 1001, 40001])
def test_swiglu_of_far_negative_gates(device, dtype, cols):
    """Gates whose divisor 1 + exp(-g) is next to fp32's largest number (its reciprocal a subnormal
    one), beside an ``up`` that makes the product a normal one: values as near as anywhere, and
    from where exp(-g) is infinite zeros, as elementary operations have them."""
    at = torch.tensor([-60.0, -69.0, -70.0, -80.0, -87.0, -87.3, -87.5, -88.0, -88.5, -88.7], device=device).to(dtype)
    gate = at[:, None].expand(-1, cols).contiguous()
    up = torch.linspace(-1, 1, cols, device=device).mul(3e4 if dtype == torch.float16 else 1e30).to(dtype).expand(len(at), -1)
    q, scale = fused_swiglu_int8(gate, up)
    g64 = gate.double()
    y = g64 / (1 + torch.exp(-g64)) * up.double()
    assert (y.abs().amax(-1) >= SMALLEST).all()
    _check(q, scale, y, 7 * U, 9 * U, f"far {dtype}")
    gone = torch.full_like(gate[:1], -89.0)
    q, scale = fused_swiglu_int8(gone, up[:1])
    assert not q.any() and not scale.any()
    gone[0, cols // 2] = float("-inf")  # -inf / inf
    q, scale = fused_swiglu_int8(gone, up[:1])
    assert torch.isnan(scale).all() and not q.any()


def _elementary_swiglu(gate, up):
    g = gate.float()
    return (g / (1 + torch.exp(-g)) * up.float()).contiguous()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(333, 2051), (65, 14336), (3, 40001)])
def test_swiglu_is_what_elementary_operations_give(device, dtype, rows, cols):
    """Bit for bit, on rows as a projection leaves them: q and scale of ``g / (1 + exp(-g)) * u``, every
    operation rounded to fp32, through ``quantize_int8``; some gates far below zero."""
    g = torch.Generator(device=device).manual_seed(cols)
    gate, up = 3 * _rand(g, (rows, cols), dtype, device), _rand(g, (rows, cols), dtype, device)
    gate[:, ::97] = (torch.rand(gate[:, ::97].shape, generator=g, device=device) * -90).to(dtype)
    for a, b in zip(fused_swiglu_int8(gate, up), quantize_int8(_elementary_swiglu(gate, up))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("up", [1.0, 3.0, -1e4, 1e30])
def test_every_gate_is_what_elementary_operations_give(device, dtype, up):
    """Rows of one value, so that the scale is the value's magnitude over 127 and shows its last bits:
    every 16-bit gate, and fp32 gates all over the range."""
    if dtype == torch.float32:
        gen = torch.Generator(device=device).manual_seed(1)
        spans = [(-105, -86), (-90, -60), (-60, 0), (-1, 1), (0, 90)]
        gate = torch.cat([lo + (hi - lo) * torch.rand(1 << 20, generator=gen, device=device) for lo, hi in spans])
    else:
        gate = torch.arange(1 << 16, dtype=torch.int32, device=device).to(torch.int16).view(dtype)
    gate = gate[:, None].contiguous()
    up = torch.full_like(gate, min(up, 6e4) if dtype == torch.float16 else up)
    for a, b in zip(fused_swiglu_int8(gate, up), quantize_int8(_elementary_swiglu(gate, up))):
        assert torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0))
        assert torch.equal(torch.isnan(a), torch.isnan(b))


@pytest.mark.parametrize("cols", [64, 1003, 16384, 40001])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_sum_in_place_of_rows_whose_squares_leave_fp32(device, cols, into):
    """The sum over one of its addends, in rows whose squares are summed again after it is written."""
    from slipstream_amd import _ffi

    g = torch.Generator(device=device).manual_seed(cols)
    sizes = torch.tensor([1.0, 2.0**70, 0.0, 2.0**-70, 2.0**100], device=device)[:, None]
    x, r = ((torch.randn(5, cols, generator=g, device=device) * sizes).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(cols, device=device, dtype=torch.bfloat16)
    want = fused_rmsnorm_int8(x, w, r, 0.0)
    _check(*want[:2], _norm64(x, w, r, 0.0)[0], 0.0, _norm_scale_err(cols), f"far {cols}")
    q = torch.empty((5, cols), dtype=torch.int8, device=device)
    scale = torch.empty(5, device=device)
    s = r if into == "residual" else x
    _ffi.check(_ffi.lib().ss_rmsnorm_int8(x.data_ptr(), r.data_ptr(), w.data_ptr(), q.data_ptr(), scale.data_ptr(),
                                          s.data_ptr(), 5, cols, cols, cols, 0.0, _ffi.dtype_code(x.dtype),
                                          _ffi.stream_ptr(device)), "norm")
    assert torch.equal(q, want[0]) and torch.equal(scale, want[1]) and torch.equal(s, want[2])
