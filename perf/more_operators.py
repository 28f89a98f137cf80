"""The operators around a cache of latents, call by call: rows quantized to 8-bit floating point
with a scale for every 128 values, the product that reads them, the latent cache's write, and
attention over latents in its absorbed form (straight from the pages) and its expanded form (keys
and values projected from the latents beforehand).

``run`` computes an operator with elementary torch operations, or (``own``) through this
framework's entry points, on the same inputs; ``exact`` gives the result in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128  # values that share a scale
TOP = 448.0  # the largest e4m3 value
SMALLEST = TOP * 2.0**-126  # blocks whose largest magnitude is below this are zeros
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # the attention's output ahead of its projection, for a decode batch of an odd size
        {"name": "rows_decodes", "kind": "rows", "m": 197, "k": 4096, "dtype": "bf16"},
        # the down projection's input for every token of a packed step
        {"name": "rows_step", "kind": "rows", "m": 2240, "k": 14336, "dtype": "bf16"},
        # one sequence's decode through the stacked gate and up projections: every weight read for one token
        {"name": "gemm_token", "kind": "gemm", "m": 1, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # every token of a packed step (4 chunks of 512 and 192 decodes) through gate and up
        {"name": "gemm_step", "kind": "gemm", "m": 2240, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # nothing is a multiple of anything: rows that start at any byte, blocks cut short, results in fp32
        {"name": "gemm_odd", "kind": "gemm", "m": 333, "n": 4999, "k": 2051, "dtype": "fp32", "bias": True},
        # the cache's write for a decode batch with an eighth of the heads, and for a packed step with all of
        # them and some padding
        {"name": "write_decodes", "kind": "write", "tokens": 256, "padding": 0, "heads": 16, "latent": 512, "rope": 64,
         "block": 16, "dtype": "bf16"},
        {"name": "write_step", "kind": "write", "tokens": 2240, "padding": 67, "heads": 128, "latent": 512, "rope": 64,
         "block": 64, "dtype": "bf16"},
        # a few chats, an eighth of the heads: latency
        {"name": "absorbed_chats", "kind": "absorbed", "decodes": 8, "median": 256, "longest": 512, "chunks": 0,
         "chunk": 0, "prior": 0, "heads": 16, "latent": 512, "rope": 64, "block": 16, "dtype": "fp16", "lengths": 1},
        # a large ragged decode batch with every head on the card
        {"name": "absorbed_decodes", "kind": "absorbed", "decodes": 256, "median": 1024, "longest": 8192, "chunks": 0,
         "chunk": 0, "prior": 0, "heads": 128, "latent": 512, "rope": 64, "block": 16, "dtype": "bf16", "lengths": 2},
        # a packed step: chunks of a prompt over what is cached, beside decodes
        {"name": "absorbed_step", "kind": "absorbed", "decodes": 192, "median": 1024, "longest": 4096, "chunks": 4,
         "chunk": 512, "prior": 4096, "heads": 16, "latent": 512, "rope": 64, "block": 64, "dtype": "bf16", "lengths": 3},
        # a follow-up question of a chat: few tokens over a short context
        {"name": "expanded_turn", "kind": "expanded", "chunks": 1, "chunk": 77, "prior": 512, "heads": 16, "nope": 128,
         "rope": 64, "v": 128, "dtype": "fp16", "lengths": 4},
        # chunks of long prompts over their context, every head on the card
        {"name": "expanded_chunks", "kind": "expanded", "chunks": 4, "chunk": 512, "prior": 4096, "heads": 128,
         "nope": 128, "rope": 64, "v": 128, "dtype": "bf16", "lengths": 5},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _width(rng, lo: int, hi: int) -> int:
    """A row length: mostly whole 128s, at times whole 16s or any number."""
    w = _log_int(rng, lo, hi)
    step = rng.choice([128, 128, 128, 16, 1])
    return max(step, w // step * step)


def draw(rng) -> dict:
    kind = rng.choice(["rows", "gemm", "gemm", "write", "absorbed", "absorbed", "expanded"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads = rng.choice([8, 14, 16, 16, 32, 64, 128, 128])
    if kind == "rows":
        return {"kind": kind, "m": _log_int(rng, 1, 2240), "k": _width(rng, 512, 14336),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "gemm":
        k = _width(rng, 512, 14336)
        n = _width(rng, 512, min(28672, 4096 * 28672 // k))
        return {"kind": kind, "m": _log_int(rng, 1, 2240), "n": n, "k": k,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "bias": rng.random() < 0.4}
    latent, block = rng.choice([512, 512, 512, 256]), rng.choice([16, 16, 32, 64])
    if kind == "write":
        tokens = _log_int(rng, 1, 2240)
        return {"kind": kind, "tokens": tokens, "padding": rng.choice([0, tokens // 7]), "heads": heads,
                "latent": latent, "rope": 64, "block": block, "dtype": dtype}
    if kind == "absorbed":
        chunks = rng.choice([0, 0, 1, 2])
        return {"kind": kind, "decodes": _log_int(rng, 1, 256) if chunks == 0 else rng.choice([0, 7, 64]),
                "median": _log_int(rng, 16, 1024), "longest": _log_int(rng, 1024, 8192), "chunks": chunks,
                "chunk": _log_int(rng, 2, max(2, 4096 // heads)) if chunks else 0,
                "prior": _log_int(rng, 1, 4096) if chunks else 0, "heads": heads, "latent": latent, "rope": 64,
                "block": block, "dtype": dtype, "lengths": rng.randrange(1 << 16)}
    return {"kind": kind, "chunks": rng.choice([1, 1, 2, 4]), "chunk": _log_int(rng, 2, 512),
            "prior": _log_int(rng, 1, 4096), "heads": heads, "nope": 128, "rope": 64, "v": 128, "dtype": dtype,
            "lengths": rng.randrange(1 << 16)}


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """Query and context lengths of a case's sequences: decodes first, then chunks."""
    rng = random.Random(case["lengths"])
    ql, cl = [], []
    for _ in range(case.get("decodes", 0)):
        ql.append(1)
        cl.append(min(case["longest"], max(1, round(case["median"] * math.exp(rng.gauss(0, 1))))))
    for i in range(case["chunks"]):
        q = case["chunk"] - (i if i < case["chunk"] - 1 else 0)  # the last parts of prompts are of any length
        ql.append(q)
        cl.append(q + rng.randint(0, case["prior"]))
    return ql, cl


def _pairs(case: dict) -> int:
    return sum(q * (c - q) + q * (q + 1) // 2 for q, c in zip(*_lens(case)))


# ---- inputs --------------------------------------------------------------------------


def _activations(gen, m: int, k: int, dtype: torch.dtype) -> torch.Tensor:
    """Rows of differing sizes in which a few channels are an order of magnitude larger, as the
    hidden states of a language model have them."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    channel = torch.rand(k, generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn((m, 1), generator=gen, device="cuda"))
    return (x * torch.where(channel < 0.004, 12.0, 1.0) * size).to(dtype)


def _in_blocks(x: torch.Tensor) -> torch.Tensor:
    """``[m, k]`` -> ``[m, blocks, 128]``, zeros behind the last column."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    return torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)


def _fp8_blocks(x: torch.Tensor, top: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 blocks and their largest magnitudes -> e4m3 blocks and their scales."""
    live = top >= SMALLEST
    q = torch.where(live, x * (TOP / torch.where(live, top, 1.0)), 0.0)
    return q.to(torch.float8_e4m3fn), torch.where(live, top / TOP, 0.0)


def _fp8_weight(gen, n: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 ``[n, k]`` with a scale for each 128 x 128 values."""
    w = torch.randn((n, k), generator=gen, device="cuda") * k**-0.5
    w *= torch.exp(0.3 * torch.randn((n, 1), generator=gen, device="cuda"))
    nb = -(-n // BLOCK)
    b = _in_blocks(torch.nn.functional.pad(w, (0, 0, 0, nb * BLOCK - n)))  # [nb * 128, kb, 128]
    b = b.view(nb, BLOCK, b.shape[1], BLOCK)
    q, scale = _fp8_blocks(b, b.abs().amax(dim=(1, 3), keepdim=True))
    return q.view(nb * BLOCK, -1)[:n, :k].contiguous(), scale.view(nb, -1).contiguous()


def _randn(gen, shape, dtype: torch.dtype, std: float) -> torch.Tensor:
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _pages(gen, cl: list[int], block: int) -> tuple[torch.Tensor, int]:
    """Block tables that hand out a pool a fifth larger than needed in random order, and its size."""
    need = [-(-c // block) for c in cl]
    pool = sum(need) + sum(need) // 5 + 1
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((len(cl), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at : at + n]
        at += n
    return tables, pool


def _starts(lens: list[int]) -> torch.Tensor:
    return torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)


def _angles(gen, tokens: int, rope: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    at = torch.randint(0, 8192, (tokens, 1), generator=gen, device="cuda").double()
    a = at * 10000.0 ** (-torch.arange(0, rope, 2, device="cuda").double() / rope)
    a = torch.cat([a, a], dim=1)
    return a.cos().to(dtype), a.sin().to(dtype)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    state = {"case": case, "dtype": dtype}
    if kind == "rows":
        state["x"] = _activations(gen, case["m"], case["k"], dtype)
    elif kind == "gemm":
        b = _in_blocks(_activations(gen, case["m"], case["k"], torch.float32))
        q, scale = _fp8_blocks(b, b.abs().amax(dim=2, keepdim=True))
        state["q"] = q.view(case["m"], -1)[:, : case["k"]].contiguous()
        # the scales of a block of columns follow each other, as the quantization leaves them
        state["scale"] = scale.squeeze(2).t().contiguous().t()
        state["qweight"], state["w_scale"] = _fp8_weight(gen, case["n"], case["k"])
        state["bias"] = _randn(gen, (case["n"],), dtype, 1.0) if case["bias"] else None
    elif kind == "write":
        t, h, r, d = case["tokens"], case["heads"], case["latent"], case["rope"]
        # as the projections leave them: a query's parts side by side, the latent and its key too
        state["q"] = _randn(gen, (t, h, 128 + d), dtype, 1.0)
        state["rows"] = _randn(gen, (t, r + d), dtype, 2.0)
        state["cos"], state["sin"] = _angles(gen, t, d, dtype)
        state["weight"] = (1 + 0.1 * torch.randn(r, generator=gen, device="cuda")).to(dtype)
        blocks = -(-t // case["block"]) + t // (5 * case["block"]) + 1
        state["cache"] = _randn(gen, (1, blocks, case["block"], r + d), dtype, 0.5)
        slots = torch.randperm(blocks * case["block"], generator=gen, device="cuda")[:t]
        if case["padding"]:
            slots[t - case["padding"] :] = -1
        state["slots"] = slots
    elif kind == "absorbed":
        ql, cl = _lens(case)
        h, r, d = case["heads"], case["latent"], case["rope"]
        state["tables"], pool = _pages(gen, cl, case["block"])
        state["cache"] = _randn(gen, (1, pool, case["block"], r + d), dtype, 1.0)
        state["q"] = _randn(gen, (sum(ql), h, r + d), dtype, 1.0)
        state["cu"], state["ctx"] = _starts(ql), torch.tensor(cl, dtype=torch.int32, device="cuda")
        state["longest"], state["scale"] = max(ql), 2.0 * (r + d) ** -0.5
    else:
        ql, cl = _lens(case)
        h, n, d, v = case["heads"], case["nope"], case["rope"], case["v"]
        state["q"] = _randn(gen, (sum(ql), h, n + d), dtype, 1.0)
        state["kv"] = _randn(gen, (sum(cl), h, n + v), dtype, 1.0)
        state["rows"] = _randn(gen, (sum(cl), 512 + d), dtype, 1.0)  # gathered latents; their keys are read here
        state["cu"], state["cu_ctx"] = _starts(ql), _starts(cl)
        state["longest"], state["scale"] = max(ql), 2.0 * (n + d) ** -0.5
    return state


# ---- the operators in elementary operations --------------------------------------------


def _turned(x: torch.Tensor) -> torch.Tensor:
    a, b = x.chunk(2, dim=-1)
    return torch.cat([-b, a], dim=-1)


def _softmax(s: torch.Tensor, hidden: int) -> torch.Tensor:
    """Over the last dimension of fp32 scores ``[.., queries, keys]``; query j sees the first
    ``keys - hidden + 1 + j`` keys."""
    tq, tk = s.shape[-2:]
    if tq > 1:
        key = torch.arange(tk, device=s.device)
        s = s.masked_fill(key > torch.arange(tq, device=s.device)[:, None] + (tk - hidden), -math.inf)
    e = torch.exp(s - s.amax(dim=-1, keepdim=True))
    return e / e.sum(dim=-1, keepdim=True)


def _plain_absorbed(state: dict) -> torch.Tensor:
    case, q = state["case"], state["q"]
    r = case["latent"]
    pages = state["cache"][0]
    out = torch.empty((*q.shape[:2], r), dtype=q.dtype, device=q.device)
    at = 0
    for i, (tq, tk) in enumerate(zip(*_lens(case))):
        n = -(-tk // case["block"])
        keys = pages[state["tables"][i, :n].long()].reshape(-1, pages.shape[2])[:tk].float()
        s = (q[at : at + tq].float().reshape(-1, keys.shape[1]) @ keys.t()).view(tq, -1, tk) * state["scale"]
        p = _softmax(s.transpose(0, 1), tq).transpose(0, 1)
        out[at : at + tq] = (p.reshape(-1, tk) @ keys[:, :r]).view(tq, -1, r).to(q.dtype)
        at += tq
    return out


def _plain_expanded(state: dict) -> torch.Tensor:
    case, q = state["case"], state["q"]
    n, v, r = case["nope"], case["v"], state["rows"].shape[1] - case["rope"]
    out = torch.empty((*q.shape[:2], v), dtype=q.dtype, device=q.device)
    at = ck = 0
    for tq, tk in zip(*_lens(case)):
        qs = q[at : at + tq].float().transpose(0, 1)  # [h, tq, n + d]
        kv = state["kv"][ck : ck + tk].float().transpose(0, 1)
        rope = state["rows"][ck : ck + tk, r:].float()
        s = torch.matmul(qs[..., :n], kv[..., :n].transpose(1, 2)) + torch.matmul(qs[..., n:], rope.t())
        p = _softmax(s * state["scale"], tq)
        out[at : at + tq] = torch.matmul(p, kv[..., n:]).transpose(0, 1).to(q.dtype)
        at, ck = at + tq, ck + tk
    return out


def _plain(state: dict):
    case, dtype, kind = state["case"], state["dtype"], state["case"]["kind"]
    if kind == "rows":
        b = _in_blocks(state["x"].float())
        top = b.abs().amax(dim=2, keepdim=True)
        live = top >= SMALLEST
        # in 64 bits: values halfway between two of the type's are common (x and top have few bits)
        q = torch.where(live, b.double() * TOP / torch.where(live, top, 1.0).double(), 0.0)
        # e4m3 has three bits behind the first one, from 2^-6 down those of 2^-6
        spacing = torch.exp2(torch.frexp(q).exponent.clamp_min(-5) - 4.0)
        q = (torch.round(q / spacing) * spacing).float()
        scale = torch.where(live, top / TOP, 0.0)
        return (q * scale).view(case["m"], -1)[:, : case["k"]], scale.squeeze(2)
    if kind == "gemm":
        k, n = case["k"], case["n"]
        x = (_in_blocks(state["q"].float()) * state["scale"].unsqueeze(2)).flatten(1)[:, :k]
        w = _in_blocks(state["qweight"].float()) * state["w_scale"].repeat_interleave(BLOCK, 0)[:n].unsqueeze(2)
        y = x @ w.flatten(1)[:, :k].t()
        return (y if state["bias"] is None else y + state["bias"].float()).to(dtype)
    if kind == "write":
        r, cos, sin = case["latent"], state["cos"].float(), state["sin"].float()
        c, k = state["rows"][:, :r].float(), state["rows"][:, r:].float()
        c = c * torch.rsqrt(c.square().mean(dim=-1, keepdim=True) + EPS) * state["weight"].float()
        row = torch.cat([c, k * cos + _turned(k) * sin], dim=1).to(dtype)
        written = case["tokens"] - case["padding"]
        state["cache"].view(-1, row.shape[1])[state["slots"][:written]] = row[:written]
        q = state["q"][..., 128:].float()
        return (q * cos[:, None] + _turned(q) * sin[:, None]).to(dtype), state["cache"]
    return _plain_absorbed(state) if kind == "absorbed" else _plain_expanded(state)


# ---- one pass ----------------------------------------------------------------------------


def _own(state: dict):
    from slipstream_amd import kernels

    case, dtype, kind = state["case"], state["dtype"], state["case"]["kind"]
    if kind == "rows":
        q, scale = kernels.quantize_fp8(state["x"])
        whole = case["k"] // BLOCK * BLOCK
        y = torch.empty(q.shape, dtype=torch.float32, device=q.device)  # the values that the rows stand for
        torch.mul(q[:, :whole].unflatten(1, (-1, BLOCK)).float(), scale[:, : whole // BLOCK, None],
                  out=y[:, :whole].unflatten(1, (-1, BLOCK)))
        if whole < case["k"]:
            y[:, whole:] = q[:, whole:].float() * scale[:, -1:]
        return y, scale
    if kind == "gemm":
        return kernels.fp8_gemm(state["q"], state["scale"], state["qweight"], state["w_scale"], state["bias"], dtype)
    if kind == "write":
        r, rows = case["latent"], state["rows"]
        q = kernels.latent_rope_and_cache(state["q"][..., 128:], rows[:, :r], rows[:, r:], state["cos"], state["sin"],
                                          state["cache"], state["slots"], 0, case["block"], state["weight"], EPS)
        return q, state["cache"]
    if kind == "absorbed":
        if state["longest"] == 1:
            out = kernels.latent_attention_decode(state["q"].unsqueeze(2), state["cache"], state["tables"], state["ctx"],
                                                  0, state["scale"], case["block"], case["latent"])
            return out.squeeze(1)
        return kernels.latent_attention_varlen(state["q"], state["cache"], state["tables"], state["cu"], state["ctx"], 0,
                                               state["scale"], case["block"], state["longest"], case["latent"])
    k_rope = state["rows"][:, state["rows"].shape[1] - case["rope"] :]
    return kernels.latent_attention_expanded(state["q"], state["kv"], k_rope, state["cu"], state["cu_ctx"],
                                             state["scale"], state["longest"])


def run(state: dict):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without, and its result in 64 bits ------------------------------


def work(case: dict) -> dict:
    es, kind = BYTES[case["dtype"]], case["kind"]
    if kind == "rows":
        m, k = case["m"], case["k"]
        return {"bytes": es * m * k + m * k + 4 * m * -(-k // BLOCK), "flops": 3.0 * m * k}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // BLOCK)
        return {"bytes": m * k + n * k + es * m * n + 4 * blocks * (m + -(-n // BLOCK)) + (es * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if kind == "write":
        t, h, r, d = case["tokens"] - case["padding"], case["heads"], case["latent"], case["rope"]
        return {"bytes": es * (t * 2 * (r + d) + case["tokens"] * 2 * (h * d + d) + r) + 8 * case["tokens"],
                "flops": 4.0 * case["tokens"] * (h * d + r + d)}
    ql, cl = _lens(case)
    h, pairs = case["heads"], _pairs(case)
    if kind == "absorbed":
        r, d = case["latent"], case["rope"]
        return {"bytes": es * (sum(cl) * (r + d) + sum(ql) * h * (2 * r + d)) + 4 * sum(-(-c // case["block"]) for c in cl),
                "flops": 2.0 * pairs * h * (2 * r + d)}
    n, d, v = case["nope"], case["rope"], case["v"]
    return {"bytes": es * (sum(cl) * (h * (n + v) + d) + sum(ql) * h * (n + d + v)), "flops": 2.0 * pairs * h * (n + d + v)}


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    f8, kind = torch.float64, case["kind"]

    def spread(unit, k):  # a value for each column from one for each block of columns
        return unit.to(f8)[:, torch.arange(k, device=unit.device) // BLOCK]

    if kind == "rows":
        x, k = st["x"].to(f8), case["k"]
        peaks = torch.stack([c.abs().max(dim=1).values for c in x.split(BLOCK, dim=1)], dim=1)
        unit = torch.where(peaks >= SMALLEST, peaks / TOP, torch.zeros_like(peaks))
        wide = spread(unit, k)
        # one division: a rounded unit would move the values that lie halfway between two of the type's
        v = torch.where(wide > 0, x * TOP / spread(peaks, k).clamp_min(1e-300), torch.zeros_like(x))
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)  # e4m3: three bits behind the first
        return torch.round(v / step) * step * wide, unit
    if kind == "gemm":
        x = st["q"].to(f8) * spread(st["scale"], case["k"])
        w = st["qweight"].to(f8) * spread(st["w_scale"], case["k"])[torch.arange(case["n"], device="cuda") // BLOCK]
        y = torch.matmul(x, w.t())
        return y if st["bias"] is None else y + st["bias"].to(f8)
    if kind == "write":
        cos, sin, r, half = st["cos"].to(f8), st["sin"].to(f8), case["latent"], case["rope"] // 2

        def rotated(v, cos, sin):
            lo, hi = v[..., :half], v[..., half:]
            return torch.cat([lo * cos[..., :half] - hi * sin[..., :half], hi * cos[..., half:] + lo * sin[..., half:]], -1)

        rows = st["rows"].to(f8)
        c = rows[:, :r]
        c = c * st["weight"].to(f8) / torch.sqrt(torch.sum(c * c, dim=1, keepdim=True) / r + EPS)
        cache = st["cache"].to(f8)
        flat = cache.view(-1, cache.shape[-1])
        use = st["slots"] >= 0
        flat[st["slots"][use]] = torch.cat([c, rotated(rows[:, r:], cos, sin)], dim=1)[use]
        return rotated(st["q"][..., 128:].to(f8), cos.unsqueeze(1), sin.unsqueeze(1)), cache
    ql, cl = _lens(case)
    starts = [sum(ql[:i]) for i in range(len(ql))]
    result = torch.zeros((sum(ql), case["heads"], case["latent"] if kind == "absorbed" else case["v"]), dtype=f8, device="cuda")

    def weights(score, b):  # [heads, queries, keys] of sequence b
        last = cl[b] - ql[b] + torch.arange(ql[b], device="cuda").view(-1, 1)  # the last key that a query sees
        score[:, torch.arange(cl[b], device="cuda").view(1, -1) > last] = -math.inf
        return torch.softmax(score, dim=2)

    if kind == "absorbed":
        for b, first in enumerate(starts):
            i = torch.arange(cl[b], device="cuda")
            slot = st["tables"][b][i // case["block"]].long() * case["block"] + i % case["block"]
            key = st["cache"].view(-1, st["cache"].shape[-1])[slot].to(f8)
            qs = st["q"][first : first + ql[b]].to(f8).permute(1, 0, 2)
            p = weights(torch.matmul(qs, key.t()) * st["scale"], b)
            result[first : first + ql[b]] = torch.matmul(p, key[:, : case["latent"]]).permute(1, 0, 2)
        return result
    offset = 0
    for b, first in enumerate(starts):
        rope = st["rows"][offset : offset + cl[b], -case["rope"] :].to(f8)
        for h in range(case["heads"]):
            kv = st["kv"][offset : offset + cl[b], h].to(f8)
            key = torch.cat([kv[:, : case["nope"]], rope], dim=1)
            score = torch.matmul(st["q"][first : first + ql[b], h].to(f8), key.t()) * st["scale"]
            result[first : first + ql[b], h] = torch.matmul(weights(score.unsqueeze(0), b)[0], kv[:, case["nope"] :])
        offset += cl[b]
    return result
