"""The W8A8 product against its formula in 64 bits, and the int8 MLP that runs it.

The integer sums are exact on both sides (doubles hold them). What is left are the roundings
of ``fma(sum * x_scale, w_scale, bias)``: the sum to fp32, the first product and the fused second
one, each 2^-24 of the value it rounds (of the value without and with the bias), and the one to
the output's type, half its eps.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from slipstream_amd import _ffi
from slipstream_amd.kernels import fused_rmsnorm_int8, fused_swiglu_int8, quantize_int8, w8a8_gemm
from slipstream_amd.quantized import W8A8Linear, W8A8MLP, quantize_weight_int8

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _case(device, m, n, k, seed=0, bias=None, full=False):
    g = torch.Generator(device=device).manual_seed(seed + 7 * m + 11 * n + 13 * k)
    low = -128 if full else -127
    q = torch.randint(low, 128, (m, k), generator=g, device=device, dtype=torch.int8)
    w = torch.randint(low, 128, (n, k), generator=g, device=device, dtype=torch.int8)
    xs = 0.001 + 0.02 * torch.rand(m, generator=g, device=device)
    ws = 1e-4 + 2e-4 * torch.rand(n, generator=g, device=device)
    b = torch.randn(n, generator=g, device=device).to(bias) if bias is not None else None
    return q, xs, w, ws, b


def _reference(q, xs, w, ws, b):
    y = (q.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    return y if b is None else y + b.double()


def _check(out, q, xs, w, ws, b, what=""):
    ref = _reference(q, xs, w, ws, b)
    assert out.shape == ref.shape, what
    plain = ref if b is None else ref - b.double()
    fp32 = 3 * U * plain.abs() + U * ref.abs()
    tol = 1.001 * (fp32 + HALF_STEP[out.dtype] * (ref.abs() + fp32)) + 1e-30
    if out.dtype == torch.float16:
        tol = tol + 2.0**-25  # half a subnormal step
    off = (out.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by {off[bad].max().item():.3e}, first {bad.nonzero()[0].tolist()}"


# every tile and its edges in m, n and k, in each output type
SHAPES = [(1, 1, 1), (1, 16, 16), (1, 17, 64), (2, 5, 3), (3, 33, 127), (4, 100, 128), (7, 63, 129), (8, 64, 192), (15, 250, 1008),
          (16, 256, 1024), (17, 257, 1040), (31, 1152, 896), (33, 96, 4864), (48, 1000, 2048), (63, 511, 511),
          (64, 512, 512), (65, 513, 528), (77, 1003, 1001), (96, 128, 4096), (127, 384, 144), (128, 640, 2064),
          (129, 130, 1936), (192, 2048, 512), (197, 4096, 1024), (255, 257, 640), (256, 256, 256), (257, 300, 272),
          (333, 999, 2051), (500, 1536, 1152), (1, 4096, 14336), (5, 28672, 512), (40, 4096, 14336), (300, 256, 16384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(device, m, n, k, dtype):
    bias = dtype if (m + n) % 2 else None
    args = _case(device, m, n, k, bias=bias)
    _check(w8a8_gemm(*args, out_dtype=dtype), *args, f"{m} x {n} x {k}")


# sizes at which each compiled kernel is the one that runs, whole 16-byte results and others: the
# stream kernel's tiles (16-row tiles of tokens, of channels, waves) and the tile kernel's (tokens x
# channels), these also with k split over workgroups
VARIANTS = [
    ("stream 1 1 2", [(33, 8480, 944), (33, 9383, 912)]), ("stream 1 1 4", [(1, 8552, 912), (7, 8425, 912)]),
    ("stream 1 1 8", [(1, 496, 1104), (13, 497, 1104)]), ("stream 1 2 2", [(35, 9832, 944), (36, 9671, 976)]),
    ("stream 1 2 4", [(1, 17168, 992), (10, 17527, 912)]), ("stream 1 2 8", [(67, 840, 1808), (34, 1463, 2016)]),
    ("stream 2 1 2", [(17, 16776, 1008), (17, 18329, 912)]), ("stream 2 1 4", [(17, 4304, 1072), (17, 4651, 1104)]),
    ("stream 2 1 8", [(17, 2072, 816), (18, 2147, 800)]), ("stream 2 2 2", [(19, 25112, 960), (17, 25637, 928)]),
    ("stream 2 2 4", [(17, 13520, 928), (17, 14749, 912)]), ("stream 2 2 8", [(21, 4472, 1456), (19, 4149, 1600)]),
    ("stream 4 2 2", [(444, 2336, 4256), (346, 2699, 5616)]), ("stream 4 2 4", [(34, 5560, 3632), (33, 6051, 3296)]),
    ("stream 4 4 4", [(33, 13456, 2848), (33, 11541, 3280)]),
    ("tile 64 128", [(572, 16, 912), (526, 17, 1008)]), ("tile 96 128", [(67, 16784, 912), (75, 16765, 928)]),
    ("tile 128 128", [(106, 18112, 912), (98, 18527, 912)]), ("tile 192 128", [(141, 22520, 976), (129, 22751, 960)]),
    ("tile 256 128", [(199, 22824, 944), (203, 26691, 928)]), ("tile 128 256", [(201, 23176, 912), (196, 24009, 1008)]),
    ("tile 160 256", [(294, 24152, 960), (257, 23769, 912)]), ("tile 192 256", [(324, 22960, 912), (348, 22249, 912)]),
    ("tile 224 256", [(434, 22232, 992), (386, 23253, 976)]), ("tile 256 256", [(479, 23552, 928), (511, 21975, 928)]),
    ("split 64 128", [(634, 16, 1696), (547, 17, 1728)]), ("split 96 128", [(1414, 16, 6768), (2207, 19, 4768)]),
    ("split 128 128", [(2140, 16, 11680), (1942, 17, 12432)]), ("split 192 128", [(140, 2760, 15888), (2075, 137, 16240)]),
    ("split 256 128", [(198, 5920, 13936), (201, 5681, 14272)]), ("split 128 256", [(201, 6136, 13168), (103, 16461, 10144)]),
    ("split 160 256", [(132, 11080, 10128), (130, 5441, 15184)]), ("split 192 256", [(161, 16504, 11936), (164, 16555, 10272)]),
    ("split 224 256", [(206, 11032, 13328), (193, 16445, 7568)]), ("split 256 256", [(238, 16784, 12080), (233, 17321, 12560)]),
    # one token block and more than 64 MB of weights
    ("once 64 128", [(33, 22240, 3024), (33, 15457, 4368)]),
    ("once 96 128", [(65, 20216, 3344), (65, 24117, 2800)]),
    ("once 128 128", [(97, 30120, 2288), (98, 31677, 2128)]),
    ("once 192 128", [(129, 16560, 4080), (131, 20097, 3344)]),
    ("once 256 128", [(193, 26832, 2512), (194, 24409, 2752)]),
    ("once 128 256", [(98, 34984, 1984), (99, 37147, 1824)]),
    ("once 160 256", [(129, 34752, 1968), (131, 33989, 2000)]),
    ("once 192 256", [(163, 34344, 1984), (167, 33053, 2032)]),
    ("once 224 256", [(193, 33280, 2064), (195, 39979, 1680)]),
    ("once 256 256", [(225, 35896, 1872), (228, 39795, 1696)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("what,shapes", VARIANTS, ids=[v[0] for v in VARIANTS])
def test_every_kernel(device, what, shapes, dtype):
    for i, (m, n, k) in enumerate(shapes):
        args = _case(device, m, n, k, bias=torch.bfloat16 if i else None)
        _check(w8a8_gemm(*args, out_dtype=dtype), *args, f"{what}: {m} x {n} x {k}")


@pytest.mark.parametrize("m", [1, 2, 16, 17, 32, 33, 48, 49, 64, 65, 80, 100, 128, 150, 200, 256, 300, 448, 513, 1000])
@pytest.mark.parametrize("n,k", [(896, 4864), (1536, 2560)])
def test_token_counts(device, m, n, k):
    args = _case(device, m, n, k)
    _check(w8a8_gemm(*args), *args, f"m = {m}")


@pytest.mark.parametrize("m", [1, 20, 64, 128, 700])
def test_largest_sums(device, m):
    """Every product 128 * 128 at the most keys that a sum holds, and of the other sign."""
    for k in (131071, 131056):
        q = torch.full((m, k), -128, dtype=torch.int8, device=device)
        w = torch.full((18, k), -128, dtype=torch.int8, device=device)
        w[3] = 127
        one = torch.ones(18, device=device)
        out = w8a8_gemm(q, torch.ones(m, device=device), w, one, out_dtype=torch.float32)
        want = torch.full((m, 18), float(128 * 128 * k), device=device)
        want[:, 3] = float(-128 * 127 * k)
        assert torch.equal(out, want)


@pytest.mark.parametrize("m,n,k", [(9, 300, 512), (70, 300, 512), (300, 520, 1024), (5, 40, 77)])
@pytest.mark.parametrize("bias", [torch.bfloat16, torch.float16, torch.float32])
def test_bias_types_and_full_range(device, m, n, k, bias):
    """Any bias type with any output type; operands from -128."""
    args = _case(device, m, n, k, bias=bias, full=True)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _check(w8a8_gemm(*args, out_dtype=dtype), *args, f"{bias} into {dtype}")


def test_leading_dimensions(device):
    q, xs, w, ws, _ = _case(device, 12, 64, 128)
    y = w8a8_gemm(q, xs, w, ws)
    assert torch.equal(w8a8_gemm(q.view(2, 3, 2, 128), xs.view(2, 3, 2), w, ws), y.view(2, 3, 2, 64))
    one = w8a8_gemm(q[4], xs[4], w, ws)
    assert one.shape == (64,) and torch.equal(one, y[4])


@pytest.mark.parametrize("m", [3, 60, 140, 600])
def test_a_row_does_not_depend_on_its_batch(device, m):
    q, xs, w, ws, b = _case(device, m, 700, 1024, bias=torch.float32)
    y = w8a8_gemm(q, xs, w, ws, b)
    for at in {0, m // 2, m - 1}:
        assert torch.equal(w8a8_gemm(q[at : at + 1], xs[at : at + 1], w, ws, b)[0], y[at])
    half = w8a8_gemm(q, xs, w[:350], ws[:350], b[:350])
    assert torch.equal(half, y[:, :350])


@pytest.mark.parametrize("m", [1, 5, 40, 70, 200, 300])
@pytest.mark.parametrize("off", [0, 1, 4, 16])
@pytest.mark.parametrize("k", [528, 531])
def test_strides_and_alignments(device, m, off, k):
    """Operands inside wider buffers at any byte; what surrounds them is 127 and is not read in.
    (Rows that do not start on 16 bytes, or whose length is not a multiple of 16, are copied first.)"""
    n = 190
    q, xs, w, ws, _ = _case(device, m, n, k)
    want = w8a8_gemm(q, xs, w, ws, out_dtype=torch.float32)
    bq = torch.full((m, k + 48), 127, dtype=torch.int8, device=device)
    bw = torch.full((n, k + 48 + off), 127, dtype=torch.int8, device=device)
    bq[:, off : off + k] = q
    bw[:, off : off + k] = w
    vq, vw = bq[:, off : off + k], bw[:, off : off + k]
    assert torch.equal(w8a8_gemm(vq, xs, vw, ws, out_dtype=torch.float32), want)
    wide = torch.stack([xs, xs + 1], 1)[:, 0]  # scales with a stride
    assert torch.equal(w8a8_gemm(vq, wide, w.t().contiguous().t(), ws, out_dtype=torch.float32), want)
    assert torch.equal(w8a8_gemm(q[:1].expand(m, k), xs[:1].expand(m), w, ws, out_dtype=torch.float32),
                       want[:1].expand(m, n))


@pytest.mark.parametrize("m,n,k", [(1, 33, 64), (50, 70, 256), (90, 70, 256), (300, 260, 512), (20, 21, 23)])
def test_nan_and_zero_scales(device, m, n, k):
    """A row marked NaN by the quantizers is NaN in every output, and only it; a row with
    scale zero is the bias."""
    q, xs, w, ws, b = _case(device, m, n, k, bias=torch.float32)
    clean = w8a8_gemm(q, xs, w, ws, b)
    q[0] = 0
    xs[0] = float("nan")
    if m > 1:
        xs[m - 1] = 0
    y = w8a8_gemm(q, xs, w, ws, b)
    assert torch.isnan(y[0]).all()
    if m > 1:
        assert torch.equal(y[m - 1], b.to(torch.bfloat16)) and torch.equal(y[1 : m - 1], clean[1 : m - 1])


@pytest.mark.parametrize("m", [1, 40, 100, 300])
def test_zero_k(device, m):
    q, w = torch.zeros((m, 0), dtype=torch.int8, device=device), torch.zeros((9, 0), dtype=torch.int8, device=device)
    b = torch.arange(9, device=device, dtype=torch.float32)
    assert torch.equal(w8a8_gemm(q, torch.ones(m, device=device), w, torch.ones(9, device=device), b),
                       b.to(torch.bfloat16).expand(m, 9))


@pytest.mark.parametrize("m,n,k", [(1, 200, 256), (20, 72, 512), (64, 200, 256), (65, 72, 512), (200, 200, 1024),
                                   (300, 264, 512), (9, 51, 77), (90, 51, 77), (140, 2760, 15888)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_c_entry_writes_its_rows_only(device, m, n, k, dtype, pad):
    """An output with a row stride, inside a buffer, without and with the workspace (of any
    contents): every result, and nothing beside them."""
    q, xs, w, ws, _ = _case(device, m, n, k)
    want = w8a8_gemm(q, xs, w, ws, out_dtype=dtype)
    lib = _ffi.lib()
    need = _ffi.ctypes.c_int64(-1)
    code = _ffi.dtype_code(dtype)
    _ffi.check(lib.ss_w8a8_workspace_size(m, n, k, 1, 1, _ffi.ctypes.byref(need)), "size")
    for nbytes in sorted({0, max(0, need.value - 1), need.value}):
        buf = torch.full((m + 2, n + pad), 77.0, dtype=dtype, device=device)
        scratch = torch.full((nbytes + 64,), 0x5A, dtype=torch.uint8, device=device)
        _ffi.check(lib.ss_w8a8_gemm(q.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, buf[1].data_ptr(),
                                    m, n, k, k, k, n + pad, code, 0, scratch.data_ptr() if nbytes else None, nbytes,
                                    _ffi.stream_ptr(device)), "gemm")
        torch.cuda.synchronize()
        assert torch.equal(buf[1 : m + 1, :n], want), nbytes
        assert (buf[0] == 77).all() and (buf[m + 1] == 77).all() and (buf[:, n:] == 77).all()
        assert (scratch[nbytes:] == 0x5A).all()


def test_weights_past_32_bit_offsets(device):
    """A weight of 4.4 GB (an output projection's kind of shape, larger): its last rows."""
    n, k = 270_000, 16384
    w = torch.zeros((n, k), dtype=torch.int8, device=device)
    tail = torch.randint(-127, 128, (5, k), device=device, dtype=torch.int8)
    w[-5:] = tail
    ws = torch.full((n,), 1e-3, device=device)
    for m in (1, 40, 130):
        q, xs, _, _, _ = _case(device, m, 5, k)
        y = w8a8_gemm(q, xs, w, ws)
        assert torch.equal(y[:, -5:], w8a8_gemm(q, xs, tail, ws[:5])) and not y[:, :-5].any()


def test_tokens_past_32_bit_offsets(device):
    """2.2 GB of tokens and an output of 4.5 GB: the last rows."""
    m, n, k = 280_000, 8000, 8000
    q = torch.zeros((m, k), dtype=torch.int8, device=device)
    tail = torch.randint(-127, 128, (3, k), device=device, dtype=torch.int8)
    q[-3:] = tail
    xs = torch.full((m,), 1e-2, device=device)
    _, _, w, ws, _ = _case(device, 1, n, k)
    y = w8a8_gemm(q, xs, w, ws)
    assert torch.equal(y[-3:], w8a8_gemm(tail, xs[:3], w, ws)) and not y[m // 2].any()


def _dense_mlp(device, hid, inter, bias, seed):
    torch.manual_seed(seed)
    mlp = torch.nn.Module()
    mlp.gate_proj = torch.nn.Linear(hid, inter, bias=bias)
    mlp.up_proj = torch.nn.Linear(hid, inter, bias=bias)
    mlp.down_proj = torch.nn.Linear(inter, hid, bias=bias)
    return mlp.to(device=device, dtype=torch.bfloat16)


def _int8_64(y):
    top = y.abs().amax(-1, keepdim=True)
    return torch.round(y * 127 / top) * (top / 127)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m", [1, 24, 197])
def test_norm_and_mlp_together(device, m, bias):
    """A layer's second half, as it is used: the norm with the residual in int8, then the int8 MLP
    (896 -> 4864 -> 896), against the same steps in 64 bits. Only values next to a rounding's
    border differ: of bf16 in gate and up (half a step, 2^-8, of rare ones), of int8 (a step
    of rare ones), and the output's own rounding, 2^-8 at most of each value, so 2^-8 of the
    norm bounds the difference with room for the rare ones (2^-8 / sqrt(3) without them)."""
    mlp = _dense_mlp(device, 896, 4864, bias, m)
    q_mlp = W8A8MLP.from_mlp(mlp)
    g = torch.Generator(device=device).manual_seed(m)
    x, r = (torch.randn(m, 896, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(896, generator=g, device=device)).to(torch.bfloat16)
    q, scale, s = fused_rmsnorm_int8(x, w, r)
    y = q_mlp.forward_int8(q, scale)

    s64 = (x.float() + r.float()).to(torch.bfloat16).double()
    assert torch.equal(s.double(), s64)
    normed = s64 * w.double() / (s64.square().mean(-1, keepdim=True) + 1e-6).sqrt()

    def linear(lin, v):
        out = _int8_64(v) @ (lin.qweight.double() * lin.scales.double()[:, None]).T
        return out if lin.bias is None else out + lin.bias.double()

    gu = linear(q_mlp.gate_up_proj, normed).to(torch.bfloat16).double()
    h = F.silu(gu[:, :4864]) * gu[:, 4864:]
    ref = linear(q_mlp.down_proj, h)
    rel = ((y.double() - ref).norm() / ref.norm()).item()
    assert rel <= 2.0**-8, rel


def test_modules_are_their_calls(device):
    """forward is quantize_int8 and the product; the MLP's parts are the separate linears'."""
    mlp = _dense_mlp(device, 256, 512, True, 0)
    m = W8A8MLP.from_mlp(mlp)
    x = torch.randn(2, 5, 256, device=device).to(torch.bfloat16)
    gate, up, down = (W8A8Linear.from_linear(lin) for lin in (mlp.gate_proj, mlp.up_proj, mlp.down_proj))
    q, scale = quantize_int8(x)
    assert torch.equal(gate(x), w8a8_gemm(q, scale, gate.qweight, gate.scales, gate.bias))
    want = down.forward_int8(*fused_swiglu_int8(gate(x), up(x)))
    assert torch.equal(m(x), want) and m(x).shape == x.shape
    scales = m.down_proj.scales.clone()
    y = m.half()(x.to(torch.float16))
    assert y.dtype == torch.float16 and m.down_proj.bias.dtype == torch.float16
    assert torch.equal(m.down_proj.scales, scales)  # still fp32


def test_int8_mlp_is_near_the_dense_one(device):
    """What int8 costs: rows and weights within half a step of a 127th of their largest value.
    For Gaussian rows of 896 (largest about 3.2 sigma) a step is 0.025 sigma, an operand's error
    0.025 / sqrt(12) = 0.7 % of it; two operands of two products, 2 % with SwiGLU's doubling."""
    mlp = _dense_mlp(device, 896, 4864, False, 3)
    x = torch.randn(64, 896, device=device).to(torch.bfloat16)
    ref = mlp.down_proj.weight.double() @ (F.silu(mlp.gate_proj.weight.double() @ x.double().T) *
                                           (mlp.up_proj.weight.double() @ x.double().T))
    y = W8A8MLP.from_mlp(mlp)(x)
    assert ((y.double().T - ref).norm() / ref.norm()).item() < 0.03


@pytest.mark.parametrize("m", [1, 24, 130, 300])
def test_captured_graph_replays(device, m):
    """Norm and MLP captured once, replayed on new inputs with eager work (another batch, which
    may take the same memory) between the replays."""
    m_q = W8A8MLP.from_mlp(_dense_mlp(device, 512, 4096, False, m))
    w = torch.ones(512, device=device, dtype=torch.bfloat16)
    x, r = (torch.randn(m, 512, device=device).to(torch.bfloat16) for _ in range(2))

    def layer(a, b):
        q, scale, s = fused_rmsnorm_int8(a, w, b)
        return m_q.forward_int8(q, scale), s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, r)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs: neither may use what the other does
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, s = layer(x, r)
        graphs.append((graph, y, s))
    for i in range(4):
        x.copy_(torch.randn(m, 512, device=device))
        r.copy_(torch.randn(m, 512, device=device))
        want, want_s = layer(x, r)
        layer(torch.randn(2 * m, 512, device=device).to(torch.bfloat16),
              torch.randn(2 * m, 512, device=device).to(torch.bfloat16))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _, _), st in zip(graphs, streams):  # both at once
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, y, s in graphs:
            assert torch.equal(y, want) and torch.equal(s, want_s), i


def test_two_streams_at_once(device):
    """Calls that overlap on two streams, each with k split over workgroups where that is done."""
    cases = [_case(device, m, 1024, 8192, seed=i) for i, m in enumerate((100, 200))]
    want = [w8a8_gemm(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(w8a8_gemm(*c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_are_quantized_alike_on_every_device(device, dtype):
    w = torch.randn(513, 1000, generator=torch.Generator().manual_seed(3)).to(dtype)
    for on_gpu, on_cpu in zip(quantize_weight_int8(w.to(device)), quantize_weight_int8(w)):
        assert torch.equal(on_gpu.cpu(), on_cpu)


# the stream kernel with one block of more than 16 tokens and weights that pass the caches by
ONCE_STREAMS = [
    ("stream 2 1 2", [(20, 18016, 3744), (23, 41409, 1664)]), ("stream 2 1 4", [(19, 12024, 5616), (18, 11835, 5856)]),
    ("stream 2 1 8", [(20, 1984, 33872), (19, 2169, 30960)]),
    ("stream 2 2 2", [(24, 28672, 4096), (29, 38581, 1744)]), ("stream 2 2 4", [(23, 15632, 4352), (29, 10633, 6464)]),
    ("stream 2 2 8", [(20, 4336, 15712), (29, 5609, 12112)]),
    ("stream 4 2 4", [(46, 7776, 9216), (39, 8015, 8416)]), ("stream 4 4 4", [(42, 12664, 5312), (44, 11135, 6064)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("what,shapes", ONCE_STREAMS, ids=[v[0] for v in ONCE_STREAMS])
def test_streams_past_the_caches(device, what, shapes, dtype):
    for i, (m, n, k) in enumerate(shapes):
        args = _case(device, m, n, k, bias=torch.bfloat16 if i else None)
        _check(w8a8_gemm(*args, out_dtype=dtype), *args, f"{what}: {m} x {n} x {k}")
