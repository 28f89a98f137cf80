"""The latent cache's write and attention over latents, absorbed and expanded, on the GPU, against the
float64 oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import latent as ora
from slipstream_amd.kernels import (
    latent_attention_decode,
    latent_attention_expanded,
    latent_attention_varlen,
    latent_rope_and_cache,
    quantize_fp8,
)
from slipstream_amd.paged_cache import allocate_latent_cache, build_packed_step
from slipstream_amd.quantized import FP8Linear

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _f64(t):
    return t.detach().cpu().double().numpy()


def _randn(gen, *shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype).cuda()


# ---- the write -----------------------------------------------------------------------------


def _angles(gen, n, rope, dtype):
    at = torch.randint(0, 5000, (n, 1), generator=gen).double()
    a = at * 10000.0 ** (-torch.arange(0, rope, 2).double() / rope)
    a = torch.cat([a, a], dim=1)
    return a.cos().to(dtype).cuda(), a.sin().to(dtype).cuda()


def _write_error(got, want, size, rows, dtype):
    """Half a step of the type, and fp32's roundings: of a rotation three, of the norm the sum's (an eighth
    of a lane's values, its tree and the total: fewer than 2^6 + 16), halved by the root, and six more."""
    tol = HALF_STEP[dtype] * np.abs(want) + 2.0**-24 * (2**6 if rows else 4) * size + (2.0**-25 if dtype == torch.float16 else 0)
    err = np.abs(got - want)
    assert np.isfinite(got).all() and (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,r,d,bs,norm", [
    (1, 16, 512, 64, 16, True), (7, 3, 512, 64, 64, True), (33, 128, 512, 64, 16, True), (5, 2, 256, 32, 32, True),
    (9, 1, 100, 6, 5, True), (4, 0, 512, 64, 16, True), (6, 5, 1536, 64, 16, True), (11, 14, 512, 64, 16, False),
    (3, 4, 40, 0, 8, True), (2, 3, 0, 8, 4, False)])
def test_write(device, dtype, n, heads, r, d, bs, norm):
    gen = torch.Generator().manual_seed(n * 100 + heads)
    q, rows = _randn(gen, n, heads, 24 + d, dtype=dtype), _randn(gen, n, r + d, dtype=dtype, std=2.0)
    cos, sin = _angles(gen, n, d, dtype)
    weight = _randn(gen, r, dtype=dtype) if norm else None
    blocks = n // bs + 3
    cache = _randn(gen, 2, blocks, bs, r + d, dtype=dtype)
    before = cache.clone()
    slots = torch.randperm(blocks * bs, generator=gen)[:n].cuda()
    if n > 4:
        slots[2], slots[4] = -1, blocks * bs + 5  # skipped
    out = latent_rope_and_cache(q[..., 24:], rows[:, :r], rows[:, r:], cos, sin, cache, slots, 1, bs, weight, 1e-5)
    c, s = _f64(cos), _f64(sin)
    qv, kv = _f64(q)[..., 24:], _f64(rows)[:, r:]
    half = np.concatenate([np.abs(qv[..., d // 2 :]), np.abs(qv[..., : d // 2])], -1)
    _write_error(_f64(out), ora.rope(qv, c[:, None], s[:, None]), np.abs(qv) + half, False, dtype)
    flat, was = cache[1].view(-1, r + d), before[1].view(-1, r + d)
    kept = torch.ones(len(flat), dtype=torch.bool)
    for t in range(n):
        slot = int(slots[t])
        if not 0 <= slot < len(flat):
            continue
        kept[slot] = False
        lat = rows[t, :r]
        if norm:
            want = ora.rms(_f64(lat), _f64(weight), 1e-5)
            _write_error(_f64(flat[slot, :r]), want, np.abs(want), True, dtype)
        else:
            assert torch.equal(flat[slot, :r], lat)
        khalf = np.concatenate([np.abs(kv[t, d // 2 :]), np.abs(kv[t, : d // 2])])
        _write_error(_f64(flat[slot, r:]), ora.rope(kv[t], c[t], s[t]), np.abs(kv[t]) + khalf, False, dtype)
    assert torch.equal(cache[0], before[0]) and torch.equal(flat[kept.cuda()], was[kept.cuda()])


def test_write_into_given_queries(device):
    """The rotated queries go into the last columns of the absorbed ones, or back where they came from;
    cos and sin of one token for all, rows of other strides."""
    gen = torch.Generator().manual_seed(4)
    n, h, r, d = 9, 4, 512, 64
    q, rows = _randn(gen, n, h, d, dtype=torch.bfloat16), _randn(gen, n, 2, r + d, dtype=torch.bfloat16)[:, 1]
    cos, sin = (t[:1].expand(n, d) for t in _angles(gen, n, d, torch.bfloat16))
    cache = allocate_latent_cache(1, 3, 16, r, d, dtype=torch.bfloat16, device=q.device)
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    args = (rows[:, :r], rows[:, r:], cos, sin, cache, slots, 0, 16)
    want = latent_rope_and_cache(q, *args)
    absorbed = torch.zeros(n, h, r + d, dtype=q.dtype, device="cuda")
    got = latent_rope_and_cache(q, *args, out=absorbed[..., r:])
    assert torch.equal(absorbed[..., r:], want) and not absorbed[..., :r].any() and got.data_ptr() == absorbed[..., r:].data_ptr()
    latent_rope_and_cache(q, *args, out=q)
    assert torch.equal(q, want)
    odd = torch.zeros(n, h, d + 1, dtype=q.dtype, device="cuda")[..., 1:]  # not on 16 bytes
    odd.copy_(want)
    assert torch.equal(latent_rope_and_cache(odd, *args), latent_rope_and_cache(want, *args))


# ---- attention -------------------------------------------------------------------------------


def _attention_error(got, want, size, reach, dtype, dims):
    """A score is a sum of ``dims`` products in fp32 (each rounding, and the scale's, below 2^-23 of the
    largest sum of magnitudes), so a probability is off by that absolutely in the exponent; 16-bit
    probabilities are rounded (half a step; those of fp16 below 2^-14 by 2^-25 of the largest), the sum of
    the rounded ones divides; exp2 and the fp32 sums over keys: 2^-15 is ample for 8192 keys; then half a
    step of the output's type."""
    prob = 0.0 if dtype == torch.float32 else HALF_STEP[dtype]
    score = 2 * 2.0**-23 * (dims + 4) * reach
    spread = size + np.abs(want)
    tol = HALF_STEP[dtype] * np.abs(want) + (prob + score + 2.0**-15) * spread * 1.01
    if dtype == torch.float16:
        tol = tol + 2.0**-13 * size.max(axis=-1, keepdims=True)  # 4096 keys' 2^-25
    err = np.abs(got - want)
    assert np.isfinite(got).all() and (err <= tol).all(), (err - tol).max()


def _pool(gen, cl, bs, width, dtype, layers=1, std=1.0):
    need = [-(-max(c, 0) // bs) for c in cl]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    tables = torch.full((len(cl), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at : at + n]
        at += n
    return _randn(gen, layers, pool, bs, width, dtype=dtype, std=std), tables


def _check_absorbed(out, q, cache, tables, ql, cl, scale, r, dtype):
    """``q [T, H, W]``, ``out [T, H, R]``, sequence by sequence."""
    at, pages = 0, _f64(cache)
    for b, (n, c) in enumerate(zip(ql, cl)):
        rows, valid = ora.gather(pages, tables[b].numpy(), c)
        want, size, reach = ora.attend(_f64(q[at : at + n]), rows, rows[:, :r], valid, c, scale)
        _attention_error(_f64(out[at : at + n]), want, size, reach, dtype, q.shape[2])
        at += n


DECODES = [  # heads, R, Dr, block, contexts
    (16, 512, 64, 16, [1, 2, 15, 16, 17, 63, 64, 65, 129, 700]),
    (16, 512, 64, 64, [0, 1, 64, 257, 1000, 31]),
    (1, 512, 64, 16, [5, 300]),
    (14, 512, 64, 16, [33, 1, 480]),
    (128, 512, 64, 16, [1, 40, 64, 777]),
    (32, 512, 64, 32, [100, 31, 600]),
    (64, 512, 64, 64, [65, 513, 3]),
    (40, 512, 64, 16, [90, 200]),
    (16, 256, 64, 16, [1, 65, 500]),
    (128, 256, 64, 16, [31, 333]),
    (8, 512, 64, 16, [3000]),
    (5, 96, 16, 16, [40, 130]),
    (3, 512, 64, 24, [100, 23, 24]),
    (2, 512, 0, 16, [70]),
    (4, 33, 7, 5, [4, 61]),
    (16, 512, 64, 1, [37]),
    (16, 512, 64, 128, [1, 129, 500]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,r,d,bs,cl", DECODES)
def test_decode(device, dtype, heads, r, d, bs, cl):
    gen = torch.Generator().manual_seed(heads * 10 + len(cl))
    cache, tables = _pool(gen, cl, bs, r + d, dtype, layers=2)
    q = _randn(gen, len(cl), heads, 1, r + d, dtype=dtype)
    scale = 1.5 * (r + d) ** -0.5
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor(cl, dtype=torch.int32).cuda(), 1, scale, bs, r)
    assert out.shape == (len(cl), 1, heads, r) and out.dtype == dtype
    _check_absorbed(out[:, 0], q[:, :, 0], cache[1], tables, [1] * len(cl), cl, scale, r, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,r,bs,ql,extra", [
    (16, 512, 16, [1, 5, 1, 40, 0, 17], [30, 0, 0, 100, 50, 9]),
    (128, 512, 64, [3, 1, 2], [100, 64, 0]),
    (16, 512, 64, [130], [300]),
    (6, 512, 16, [33, 2], [0, 129]),
    (20, 256, 16, [9, 1], [64, 5]),
    (3, 64, 16, [7, 1, 12], [3, 70, 0]),
])
def test_packed_step(device, dtype, heads, r, bs, ql, extra):
    gen = torch.Generator().manual_seed(heads + len(ql))
    cl = [a + b for a, b in zip(ql, extra)]
    cache, tables = _pool(gen, cl, bs, r + 64, dtype)
    total = sum(ql)
    q = _randn(gen, total + 3, heads, r + 64, dtype=dtype)
    cu = torch.tensor([0] + ql).cumsum(0).to(torch.int32).cuda()
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    scale = -1.2 * (r + 64) ** -0.5 if heads == 6 else 1.2 * (r + 64) ** -0.5
    out = torch.full((total + 3, heads, r + 8), 7.0, dtype=dtype, device="cuda")[..., :r]
    got = latent_attention_varlen(q, cache, tables.cuda(), cu, ctx, 0, scale, bs, max(ql), r, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[total:] == 7).all()  # rows behind the last sequence stay
    _check_absorbed(out, q, cache[0], tables, ql, cl, scale, r, dtype)
    again = latent_attention_varlen(q, cache, tables.cuda(), cu, ctx, 0, scale, bs, 1, r)[:total]
    _check_absorbed(again, q, cache[0], tables, ql, cl, scale, r, dtype)  # whatever max_query_len says


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [16, 128])
def test_absent_pages_and_what_lies_behind_a_sequence(device, dtype, heads):
    """Absent pages and entries past the pool are masked, a sequence without any page gives zeros, a table
    narrower than the length ends it; NaN behind a sequence's end and in other pages reaches nobody."""
    gen = torch.Generator().manual_seed(8)
    r, d, bs, cl = 512, 64, 16, [50, 70, 200, 33, 64]
    cache, tables = _pool(gen, cl, bs, r + d, dtype)
    tables[1, 1], tables[2, 4], tables[2, 5] = -1, cache.shape[1] + 9, -7
    used = torch.zeros(cache.shape[1], dtype=torch.bool)
    for b, c in enumerate(cl):
        for i in range(-(-c // bs)):
            e = int(tables[b, i])
            if not 0 <= e < cache.shape[1]:
                continue
            used[e] = True
            if (i + 1) * bs > c:
                cache[0, e, c - i * bs :] = float("nan")
    cache[0, ~used.cuda()] = float("inf")
    tables[3] = -1
    cl_given = list(cl)
    cl_given[4] = 64 + 300  # more than its table holds? the table is as wide as the longest: masked entries
    q = _randn(gen, len(cl), heads, 1, r + d, dtype=dtype)
    ctx = torch.tensor(cl_given, dtype=torch.int32).cuda()
    out = latent_attention_decode(q, cache, tables.cuda(), ctx, 0, 0.05, bs, r)
    _check_absorbed(out[:, 0], q[:, :, 0], cache[0].nan_to_num(0, 0, 0), tables, [1] * 5, cl_given, 0.05, r, dtype)
    assert not out[3].any()
    negative = latent_attention_decode(q, cache, tables.cuda(), -ctx, 0, 0.05, bs, r)
    assert not negative.any()


@pytest.mark.parametrize("heads", [16, 128])
def test_queries_longer_than_the_context_see_what_there_is(device, heads):
    """The first queries of a sequence with fewer keys than queries see none: zeros."""
    gen = torch.Generator().manual_seed(9)
    cache, tables = _pool(gen, [20], 16, 576, torch.bfloat16)
    q = _randn(gen, 1, heads, 30, 576, dtype=torch.bfloat16)
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor([20], dtype=torch.int32).cuda(), 0, 0.05, 16, 512)
    _check_absorbed(out[0], q[0].transpose(0, 1), cache[0], tables, [30], [20], 0.05, 512, torch.bfloat16)
    assert not out[0, :10].any() and out[0, 10:].any()


@pytest.mark.parametrize("heads", [16, 128])
def test_a_large_score_late_in_the_context(device, heads):
    """The running maximum grows by far more than any slack, up and down, and stays exact."""
    gen = torch.Generator().manual_seed(10)
    cache, tables = _pool(gen, [900], 16, 576, torch.bfloat16, std=0.5)
    q = _randn(gen, 1, heads, 1, 576, dtype=torch.bfloat16)
    flat = tables[0, torch.arange(900) // 16].long() * 16 + torch.arange(900) % 16
    rows = cache[0].view(-1, 576)
    for at, f in ((3, -3.0), (70, 1.0), (200, 2.0), (500, 6.0), (899, 5.5)):
        rows[flat[at]] = q[0, at % heads, 0] * f / 4
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor([900], dtype=torch.int32).cuda(), 0, 0.2, 16, 512)
    _check_absorbed(out[:, 0], q[:, :, 0], cache[0], tables, [1], [900], 0.2, 512, torch.bfloat16)


def test_layouts_streams_and_broken_streams(device):
    gen = torch.Generator().manual_seed(11)
    ql, cl, r, d, bs, heads = [1, 6, 1], [40, 70, 100], 512, 64, 16, 16
    cache, tables = _pool(gen, cl, bs, r + d, torch.bfloat16)
    wide = torch.zeros(1, cache.shape[1], bs, r + d + 24, dtype=cache.dtype, device="cuda")[..., 8 : 8 + r + d]
    wide.copy_(cache)
    q = _randn(gen, 8, heads, r + d, dtype=torch.bfloat16)
    cu, ctx = torch.tensor([0, 1, 7, 8], dtype=torch.int32).cuda(), torch.tensor(cl, dtype=torch.int32).cuda()
    args = (tables.cuda(), cu, ctx, 0, 0.05, bs, 6, r)
    want = latent_attention_varlen(q, cache, *args)
    _check_absorbed(want, q, cache[0], tables, ql, cl, 0.05, r, torch.bfloat16)
    assert torch.equal(latent_attention_varlen(q, wide, *args), want)  # rows apart, on 16 bytes
    odd = torch.zeros(1, cache.shape[1], bs, r + d + 1, dtype=cache.dtype, device="cuda")[..., 1:]
    odd.copy_(cache)
    got = latent_attention_varlen(q, odd, *args)  # not on 16 bytes: the general kernel
    _check_absorbed(got, q, cache[0], tables, ql, cl, 0.05, r, torch.bfloat16)
    assert torch.equal(latent_attention_varlen(q.transpose(0, 1).contiguous().transpose(0, 1), cache, *args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = latent_attention_varlen(q, cache, tables.long().cuda(), cu.long(), ctx.long(), 0, 0.05, bs, 6, r)
    side.synchronize()
    assert torch.equal(other, want)
    # a stream past the tokens is clamped, one that runs backwards counts as empty
    past = latent_attention_varlen(q, cache, tables.cuda(), torch.tensor([0, 1, 7, 50], dtype=torch.int32).cuda(), ctx, 0,
                                   0.05, bs, 6, r)
    assert torch.equal(past, want)
    back = torch.full((8, heads, r), 3.0, dtype=q.dtype, device="cuda")
    latent_attention_varlen(q, cache, tables.cuda(), torch.tensor([-4, 1, 0, 1], dtype=torch.int32).cuda(), ctx, 0, 0.05, bs,
                            6, r, out=back)
    assert (back[1:] == 3).all() and torch.isfinite(back.float()).all()


def test_long_cache_offsets_pass_32_bits(device):
    """A pool of more than 2^31 values and 2^32 bytes, whose last pages are read."""
    r, d, bs, heads = 512, 64, 64, 16
    blocks = (1 << 32) // (bs * (r + d) * 2) + 200
    cache = torch.zeros(1, blocks, bs, r + d, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(12)
    pages = [blocks - 1, blocks // 2, blocks - 60, 0, blocks - 7]
    small = _randn(gen, 1, len(pages), bs, r + d, dtype=torch.bfloat16)
    cache[0, pages] = small[0]
    q = _randn(gen, 1, heads, 1, r + d, dtype=torch.bfloat16)
    ctx = torch.tensor([300], dtype=torch.int32).cuda()
    out = latent_attention_decode(q, cache, torch.tensor([pages], dtype=torch.int32).cuda(), ctx, 0, 0.05, bs, r)
    again = latent_attention_decode(q, small, torch.arange(5, dtype=torch.int32).view(1, 5).cuda(), ctx, 0, 0.05, bs, r)
    assert torch.equal(out, again) and again.any()


# ---- the expanded form -----------------------------------------------------------------------


def _check_expanded(out, q, kv, k_rope, ql, cl, scale, nope, dtype):
    at = ck = 0
    for n, c in zip(ql, cl):
        k = _f64(kv[ck : ck + c])
        rope = np.repeat(_f64(k_rope[ck : ck + c])[:, None], q.shape[1], axis=1)
        want, size, reach = ora.attend(_f64(q[at : at + n]), np.concatenate([k[..., :nope], rope], -1), k[..., nope:],
                                       np.ones(c, dtype=bool), c, scale)
        _attention_error(_f64(out[at : at + n]), want, size, reach, dtype, q.shape[2])
        at, ck = at + n, ck + c


EXPANDED = [  # heads, Dn, Dr, Dv, query lengths, further context
    (2, 128, 64, 128, [1, 5, 64, 0, 17], [0, 60, 3, 9, 130]),
    (3, 128, 64, 128, [130, 1], [70, 300]),
    (1, 128, 64, 128, [300], [0]),
    (2, 128, 64, 128, [257, 33], [200, 31]),
    (16, 128, 64, 128, [3, 2, 1], [500, 0, 0]),
    (2, 64, 32, 64, [40, 7], [10, 80]),
    (2, 128, 0, 128, [20], [40]),
    (3, 40, 8, 56, [9, 21], [30, 0]),
    (1, 192, 64, 512, [10], [90]),
    (2, 7, 3, 5, [4], [6]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dn,dr,dv,ql,extra", EXPANDED)
def test_expanded(device, dtype, heads, dn, dr, dv, ql, extra):
    gen = torch.Generator().manual_seed(heads + dn + len(ql))
    cl = [a + b for a, b in zip(ql, extra)]
    total, keys = sum(ql), sum(cl)
    q, kv = _randn(gen, total + 2, heads, dn + dr, dtype=dtype), _randn(gen, keys, heads, dn + dv, dtype=dtype)
    rows = _randn(gen, keys, 24 + dr, dtype=dtype)
    cu, cu_ctx = (torch.tensor([0] + n).cumsum(0).to(torch.int32).cuda() for n in (ql, cl))
    scale = (-1.5 if dn == 40 else 1.5) * (dn + dr) ** -0.5
    out = torch.full((total + 2, heads, dv + 8), 7.0, dtype=dtype, device="cuda")[..., :dv]
    got = latent_attention_expanded(q, kv, rows[:, 24:], cu, cu_ctx, scale, max(ql), out=out)
    assert got.data_ptr() == out.data_ptr() and (out[total:] == 7).all()
    _check_expanded(out, q, kv, rows[:, 24:], ql, cl, scale, dn, dtype)
    again = latent_attention_expanded(q, kv, rows[:, 24:], cu, cu_ctx, scale, 1)
    _check_expanded(again, q, kv, rows[:, 24:], ql, cl, scale, dn, dtype)  # whatever max_query_len says


def test_expanded_edges(device):
    """More queries than keys, streams that run past their ends, NaN in rows of no sequence."""
    gen = torch.Generator().manual_seed(21)
    q, kv, kr = (_randn(gen, *s, dtype=torch.bfloat16) for s in ((40, 2, 192), (90, 2, 256), (90, 64)))
    kv[20:30] = float("nan")
    kr[20:30] = float("inf")
    cu, cu_ctx = torch.tensor([0, 30, 40], dtype=torch.int32).cuda(), torch.tensor([0, 20, 20], dtype=torch.int32).cuda()
    out = latent_attention_expanded(q, kv, kr, cu, cu_ctx, 0.1, 30)
    _check_expanded(out[:30], q[:30], kv, kr, [30], [20], 0.1, 128, torch.bfloat16)
    assert not out[:10].any() and not out[30:].any()  # fewer keys than queries; no key at all
    far, far_ctx = torch.tensor([0, 30, 400], dtype=torch.int32).cuda(), torch.tensor([0, 20, 2000], dtype=torch.int32).cuda()
    clean = (kv.nan_to_num(0), kr.nan_to_num(0, 0, 0))
    past = latent_attention_expanded(q, *clean, far, far_ctx, 0.1, 30)
    _check_expanded(past, q, *clean, [30, 10], [20, 70], 0.1, 128, torch.bfloat16)


# ---- a step as a layer runs it -----------------------------------------------------------------


def _layer(gen, hidden, heads, r, dn, dr, dv):
    def linear(n, k):
        lin = torch.nn.Linear(k, n, bias=False)
        with torch.no_grad():
            lin.weight.copy_(torch.randn(n, k, generator=gen) * k**-0.5)
        return FP8Linear.from_linear(lin.to(torch.bfloat16)).cuda()

    return {"q": linear(heads * (dn + dr), hidden), "down": linear(r + dr, hidden), "out": linear(hidden, heads * dv),
            "up": linear(heads * (dn + dv), r), "norm": _randn(gen, r, dtype=torch.bfloat16)}


def test_layer_step(device):
    """A decode step and a chunk through the FP8 projections, the cache's write and both forms of the
    attention: the forms agree, and the decode replays from a graph as it runs eagerly."""
    gen = torch.Generator().manual_seed(30)
    hidden, heads, r, dn, dr, dv, bs = 256, 4, 512, 128, 64, 128, 16
    w = _layer(gen, hidden, heads, r, dn, dr, dv)
    up = (w["up"].qweight.float() * w["up"].scales.repeat_interleave(128, 0).repeat_interleave(128, 1)).to(torch.bfloat16)
    up = up.view(heads, dn + dv, r)
    wk, wv = up[:, :dn].contiguous(), up[:, dn:].transpose(1, 2).contiguous()  # [H, Dn, R], [H, R, Dv]
    scale = (dn + dr) ** -0.5
    prior, ql = [30, 0, 77], [5, 40, 1]
    cl = [a + b for a, b in zip(prior, ql)]
    cache, tables = _pool(gen, cl, bs, r + dr, torch.bfloat16)
    tables = tables.cuda()
    total = sum(ql)
    x = _randn(gen, total, hidden, dtype=torch.bfloat16)
    step = build_packed_step(tables, torch.tensor(prior, dtype=torch.int32).cuda(), torch.tensor(ql, dtype=torch.int32).cuda(),
                             bs, total, max(ql))
    cos, sin = _angles(gen, total, dr, torch.bfloat16)

    def absorbed(x, step, cos, sin):
        rows8, s8 = quantize_fp8(x)
        q = w["q"].forward_fp8(rows8, s8).view(-1, heads, dn + dr)
        rows = w["down"].forward_fp8(rows8, s8)
        qa = torch.empty((x.shape[0], heads, r + dr), dtype=x.dtype, device=x.device)
        qa[..., :r] = torch.bmm(q[..., :dn].transpose(0, 1).contiguous(), wk).transpose(0, 1)
        latent_rope_and_cache(q[..., dn:], rows[:, :r], rows[:, r:], cos, sin, cache, step.slot_mapping, 0, bs, w["norm"],
                              out=qa[..., r:])
        o = latent_attention_varlen(qa, cache, step.block_tables, step.cu_seqlens, step.context_lens, 0, scale, bs,
                                    step.max_query_len, r)
        o = torch.bmm(o.transpose(0, 1).contiguous(), wv).transpose(0, 1).reshape(-1, heads * dv)
        return w["out"](o), o, qa, q

    y, o, qa, q = absorbed(x, step, cos, sin)
    # the expanded form over the same cache: the context's latents by their slots, projected in FP8
    ctx = build_packed_step(tables, torch.zeros(3, dtype=torch.int32).cuda(), step.context_lens, bs, sum(cl), max(cl))
    rows = cache[0].view(-1, r + dr).index_select(0, ctx.slot_mapping)
    kv = w["up"](rows[:, :r]).view(-1, heads, dn + dv)
    qe = torch.cat([q[..., :dn], qa[..., r:]], dim=-1)
    e = latent_attention_expanded(qe, kv, rows[:, r:], step.cu_seqlens, ctx.cu_seqlens, scale, step.max_query_len)
    _check_expanded(e, qe, kv, rows[:, r:], ql, cl, scale, dn, torch.bfloat16)
    _check_absorbed(latent_attention_varlen(qa, cache, tables, step.cu_seqlens, step.context_lens, 0, scale, bs, 40, r), qa,
                    cache[0], tables.cpu(), ql, cl, scale, r, torch.bfloat16)
    # the latents' e4m3 rounding (2^-4) in keys and values stands between the forms: far apart would be a wrong layout
    a, b = _f64(o), _f64(e).reshape(total, -1)
    assert np.linalg.norm(a - b) < 0.1 * np.linalg.norm(b)
    # decode: captured once, replayed with other inputs between eager calls
    n = 3
    xd, cosd, sind = x[:n].clone(), cos[:n].clone(), sin[:n].clone()
    prior_d = torch.tensor(cl, dtype=torch.int32).cuda() - 1
    ones = torch.ones(n, dtype=torch.int32).cuda()

    def decode():
        return absorbed(xd, build_packed_step(tables, prior_d, ones, bs, n, 1), cosd, sind)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = decode()
    for seed in range(3):
        xd.copy_(torch.randn(n, hidden, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        prior_d.copy_(torch.tensor([33 - seed, 20 + seed, 70], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, decode())
