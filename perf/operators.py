"""The operators of the 8-bit integer linear path, call by call: rows quantized to int8 with a
scale each (alone, behind the RMS norm with the residual's addition, behind SwiGLU) and the
int8 product with a scale for each token and channel that reads them.

``run`` computes an operator with elementary torch operations, or (``own``) through this
framework's entry points, on the same inputs; ``exact`` gives the result in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
LEVELS = 127.0
SMALLEST = LEVELS * 2.0**-126  # rows whose largest magnitude is below this are zeros


def listed() -> list[dict]:
    return [
        # one sequence's decode through the stacked gate and up projections: every weight read for one token
        {"name": "gemm_token", "kind": "gemm", "m": 1, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # a few chats on a small model, q, k and v stacked with their bias: one launch's latency
        {"name": "gemm_qkv_small", "kind": "gemm", "m": 11, "n": 1152, "k": 896, "dtype": "fp16", "bias": True},
        # a decode batch of an odd size through the down projection
        {"name": "gemm_decodes", "kind": "gemm", "m": 197, "n": 4096, "k": 14336, "dtype": "bf16", "bias": False},
        # every token of a packed step (4 chunks of 512 and 192 decodes) through gate and up
        {"name": "gemm_step", "kind": "gemm", "m": 2240, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # nothing is a multiple of anything: a pruned layer's sizes, rows that start at any byte, results in fp32
        {"name": "gemm_odd", "kind": "gemm", "m": 333, "n": 4999, "k": 2051, "dtype": "fp32", "bias": True},
        # the norm before a layer's projections: one decode token, and a packed step's
        {"name": "norm_token", "kind": "norm", "m": 1, "k": 4096, "dtype": "bf16", "residual": True},
        {"name": "norm_step", "kind": "norm", "m": 2240, "k": 4096, "dtype": "bf16", "residual": True},
        # the down projection's input: a small model's decode batch, and a packed step's tokens;
        # gate and up are the halves of one projection's output
        {"name": "swiglu_small", "kind": "swiglu", "m": 11, "k": 4864, "dtype": "fp16"},
        {"name": "swiglu_step", "kind": "swiglu", "m": 2240, "k": 14336, "dtype": "bf16"},
        # the attention's output ahead of its projection, and a long prompt's rows at an odd width in fp32
        {"name": "rows_decodes", "kind": "rows", "m": 197, "k": 4096, "dtype": "bf16"},
        {"name": "rows_odd", "kind": "rows", "m": 6001, "k": 2051, "dtype": "fp32"},
        # norm, gate and up, SwiGLU and down for a small decode batch, as a layer runs them
        {"name": "mlp_batch", "kind": "mlp", "m": 24, "hidden": 4096, "inter": 14336, "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _width(rng, lo: int, hi: int) -> int:
    """A row length: mostly whole 128s, at times whole 16s or any number."""
    w = _log_int(rng, lo, hi)
    step = rng.choice([128, 128, 128, 16, 1])
    return max(step, w // step * step)


def draw(rng) -> dict:
    kind = rng.choice(["gemm", "gemm", "gemm", "norm", "swiglu", "rows", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    m = _log_int(rng, 1, 2240)
    if kind == "gemm":
        k = _width(rng, 512, 14336)
        n = _width(rng, 512, min(28672, 4096 * 28672 // k))
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.4}
    if kind == "norm":
        return {"kind": kind, "m": m, "k": _width(rng, 512, 16384), "dtype": dtype, "residual": rng.random() < 0.7}
    if kind == "swiglu":
        return {"kind": kind, "m": m, "k": _width(rng, 512, 14336), "dtype": dtype}
    if kind == "rows":
        return {"kind": kind, "m": m, "k": _width(rng, 512, 16384), "dtype": dtype}
    return {"kind": kind, "m": _log_int(rng, 1, 512), "hidden": 128 * _log_int(rng, 7, 32),
            "inter": 128 * _log_int(rng, 16, 112), "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ---- inputs --------------------------------------------------------------------------


def _activations(gen, m: int, k: int, dtype: torch.dtype) -> torch.Tensor:
    """Rows of differing sizes in which a few channels are an order of magnitude larger, as the
    hidden states of a language model have them."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    channel = torch.rand(k, generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn((m, 1), generator=gen, device="cuda"))
    return (x * torch.where(channel < 0.004, 12.0, 1.0) * size).to(dtype)


def _int8_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    top = x.abs().amax(dim=-1, keepdim=True)
    return torch.round(x * (LEVELS / top)).to(torch.int8), (top / LEVELS).squeeze(-1)


def _weight(gen, n: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _int8_rows(torch.randn((n, k), generator=gen, device="cuda") * k**-0.5)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, m, kind = DTYPES[case["dtype"]], case["m"], case["kind"]
    state = {"case": case, "dtype": dtype}
    if kind == "gemm":
        state["q"], state["scale"] = _int8_rows(_activations(gen, m, case["k"], torch.float32))
        state["qweight"], state["w_scale"] = _weight(gen, case["n"], case["k"])
        state["bias"] = torch.randn(case["n"], generator=gen, device="cuda").to(dtype) if case["bias"] else None
    elif kind == "swiglu":
        both = _activations(gen, m, 2 * case["k"], dtype)
        state["gate"], state["up"] = both[:, : case["k"]], both[:, case["k"] :]
    elif kind == "rows":
        state["x"] = _activations(gen, m, case["k"], dtype)
    else:  # norm, mlp
        k = case["hidden"] if kind == "mlp" else case["k"]
        state["x"] = _activations(gen, m, k, dtype)
        state["residual"] = _activations(gen, m, k, dtype) if kind == "mlp" or case["residual"] else None
        state["weight"] = (1 + 0.1 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        if kind == "mlp":
            state["qgate_up"], state["gate_up_scale"] = _weight(gen, 2 * case["inter"], k)
            state["qdown"], state["down_scale"] = _weight(gen, k, case["inter"])
    return state


# ---- the operators in elementary operations --------------------------------------------


def _plain_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows -> their int8 values (held in fp32) and scales."""
    top = y.abs().amax(dim=-1, keepdim=True)
    live = top >= SMALLEST
    q = torch.round(y * (LEVELS / torch.where(live, top, 1.0))) * live
    return q, torch.where(live, top / LEVELS, 0.0)


def _plain_norm(x, weight, residual):
    """The normalised rows in fp32, and x + residual in the inputs' type."""
    hidden = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    s = (x if hidden is None else hidden).float()
    return s * torch.rsqrt(s.square().mean(dim=-1, keepdim=True) + EPS) * weight.float(), hidden


def _plain_swiglu(gate, up):
    g = gate.float()
    return g / (1.0 + torch.exp(-g)) * up.float()


def _plain_gemm(q, scale, qweight, w_scale, bias, dtype):
    y = (q.float() @ qweight.float().T) * scale * w_scale
    return (y if bias is None else y + bias.float()).to(dtype)


def _plain(state: dict):
    case, dtype = state["case"], state["dtype"]
    if case["kind"] == "gemm":
        return _plain_gemm(state["q"], state["scale"][:, None], state["qweight"], state["w_scale"], state["bias"], dtype)
    if case["kind"] == "mlp":
        y, hidden = _plain_norm(state["x"], state["weight"], state["residual"])
        gu = _plain_gemm(*_plain_rows(y), state["qgate_up"], state["gate_up_scale"], None, dtype)
        h = _plain_swiglu(gu[:, : case["inter"]], gu[:, case["inter"] :])
        return _plain_gemm(*_plain_rows(h), state["qdown"], state["down_scale"], None, dtype), hidden
    hidden = None
    if case["kind"] == "norm":
        y, hidden = _plain_norm(state["x"], state["weight"], state["residual"])
    elif case["kind"] == "swiglu":
        y = _plain_swiglu(state["gate"], state["up"])
    else:
        y = state["x"].float()
    q, scale = _plain_rows(y)
    return (q * scale).to(torch.bfloat16), scale.squeeze(-1), hidden


# ---- one pass ----------------------------------------------------------------------------


def _values(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What int8 rows stand for; their eight bits are few enough for bf16."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _own(state: dict):
    from slipstream_amd.kernels import fused_rmsnorm_int8, fused_swiglu_int8, quantize_int8, w8a8_gemm

    case, dtype = state["case"], state["dtype"]
    if case["kind"] == "gemm":
        return w8a8_gemm(state["q"], state["scale"], state["qweight"], state["w_scale"], state["bias"], dtype)
    if case["kind"] == "mlp":
        q, scale, hidden = fused_rmsnorm_int8(state["x"], state["weight"], state["residual"], EPS)
        gu = w8a8_gemm(q, scale, state["qgate_up"], state["gate_up_scale"], None, dtype)
        q, scale = fused_swiglu_int8(gu[:, : case["inter"]], gu[:, case["inter"] :])
        return w8a8_gemm(q, scale, state["qdown"], state["down_scale"], None, dtype), hidden
    hidden = None
    if case["kind"] == "norm":
        q, scale, hidden = fused_rmsnorm_int8(state["x"], state["weight"], state["residual"], EPS)
    elif case["kind"] == "swiglu":
        q, scale = fused_swiglu_int8(state["gate"], state["up"])
    else:
        q, scale = quantize_int8(state["x"])
    return _values(q, scale), scale, hidden


def run(state: dict):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without, and its result in 64 bits ------------------------------


def work(case: dict) -> dict:
    m, es, kind = case["m"], BYTES[case["dtype"]], case["kind"]

    def gemm(n, k, bias=False):
        return m * k + n * k + es * m * n + 4 * (m + n) + (es * n if bias else 0), 2.0 * m * n * k

    if kind == "gemm":
        nbytes, flops = gemm(case["n"], case["k"], case["bias"])
        return {"bytes": nbytes, "flops": flops}
    if kind == "mlp":
        # the weights, the block's own inputs and outputs; what passes between its calls need not leave the chip
        h, i = case["hidden"], case["inter"]
        return {"bytes": 3 * h * i + 4 * (2 * i + h) + es * (4 * m * h + h), "flops": 6.0 * m * h * i}
    k = case["k"]
    out = m * k + 4 * m
    if kind == "norm":
        return {"bytes": es * (m * k * (3 if case["residual"] else 1) + k) + out, "flops": 8.0 * m * k}
    if kind == "swiglu":
        return {"bytes": 2 * es * m * k + out, "flops": 10.0 * m * k}
    return {"bytes": es * m * k + out, "flops": 4.0 * m * k}


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    f8, dtype, kind = torch.float64, st["dtype"], case["kind"]

    def stored(v):  # a value that the path keeps in the inputs' type, widened again
        return v.to(dtype).to(f8)

    def int8(v):
        peak = v.abs().max(dim=1, keepdim=True).values
        unit = peak / 127
        code = torch.where(peak >= SMALLEST, torch.round(v / unit.clamp_min(1e-300)), torch.zeros_like(v))
        return code, torch.where(peak >= SMALLEST, unit, torch.zeros_like(unit))

    def product(code, unit, w, w_unit):
        return torch.matmul(code.to(f8), w.to(f8).t()).mul_(unit.to(f8)).mul_(w_unit.to(f8))

    def normed():
        s = st["x"].to(f8)
        total = None
        if st["residual"] is not None:
            total = s + st["residual"].to(f8)
            s = stored(total)
        return s * st["weight"].to(f8) / torch.sqrt(torch.sum(s * s, dim=1, keepdim=True) / s.shape[1] + EPS), total

    def gated(g, u):
        return g.to(f8) * torch.sigmoid(g.to(f8)) * u.to(f8)

    if kind == "gemm":
        y = product(st["q"], st["scale"].unsqueeze(1), st["qweight"], st["w_scale"])
        return y if st["bias"] is None else y + st["bias"].to(f8)
    if kind == "mlp":
        y, total = normed()
        gu = stored(product(*int8(y), st["qgate_up"], st["gate_up_scale"]))
        return product(*int8(gated(*gu.chunk(2, dim=1))), st["qdown"], st["down_scale"]), total
    total = None
    if kind == "norm":
        y, total = normed()
    else:
        y = gated(st["gate"], st["up"]) if kind == "swiglu" else st["x"].to(f8)
    code, unit = int8(y)
    return code * unit, unit.squeeze(1), total
