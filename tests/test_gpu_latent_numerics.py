"""What attention over latents does with probabilities in 16 bits: rows that one key outweighs, and rows that many keys
far below one make up."""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_latent import _pool, _randn

from slipstream_amd.kernels import latent_attention_decode, latent_attention_expanded, latent_attention_varlen

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def _cu(n):
    return torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()


# Rows whose value is known whatever their probabilities are. "apart": one key's score is 2^18 (log2) above all
# others', and the scores are so large that its distance from their rounded maximum is a fraction of a step of the type
# away from 0: the row is that key's value. "lagging": one key is up to 2^7.8 above the one that the running maximum was
# last raised to, and all keys have the same value, which the row is then.
#
# Values have the output's type. A value's product with a probability of 11 bits or fewer is exact in fp32; sums of n
# such products and of n probabilities, and the quotient by way of a reciprocal, are off by (2 n + 4) 2^-24 altogether,
# 2^-12 at most for 2000 keys and far less where all but two probabilities vanish (as they do here: 2^-21). Half a step
# next to a value is 2^-12 (fp16) or 2^-9 (bf16) of it at least: the value comes back bit for bit.


def _scores(kind: str, n: int, at: int, dtype) -> torch.Tensor:
    s = torch.full((n,), -64.0 if kind == "apart" else -100.0)
    if kind == "apart":
        s[at] = 64.0
    else:
        s[0], s[at] = 0.0, 7.75
    return s.to(dtype).cuda()


def _factors(kind: str, heads: int, dtype) -> torch.Tensor:
    """Queries by which the heads' scores differ: other fractions of a power of two for each."""
    return ((1 if kind == "apart" else 0.5) + torch.arange(heads) / (2 * heads)).to(dtype).cuda()


SCALE = {"apart": 3000.0, "lagging": 0.6931}


def _values(kind: str, rows: torch.Tensor) -> None:
    if kind == "lagging":
        rows[:] = rows[:1]


@pytest.mark.parametrize("kind", ["apart", "lagging"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,r", [(16, 512), (32, 512), (64, 512), (128, 512), (16, 256), (128, 256)])
def test_decode_rows_of_one_value(device, kind, dtype, heads, r):
    gen = torch.Generator().manual_seed(heads + r)
    cl = [1, 33, 200, 500, 1900]
    cache, tables = _pool(gen, cl, 16, r + 64, dtype)
    flat, q = cache[0].view(-1, r + 64), torch.zeros(len(cl), heads, 1, r + 64, dtype=dtype, device="cuda")
    q[:, :, 0, r] = _factors(kind, heads, dtype)
    want = torch.zeros(len(cl), heads, r, dtype=dtype, device="cuda")
    _values(kind, flat[:, :r])
    for b, c in enumerate(cl):
        slots = (tables[b, torch.arange(c) // 16].long() * 16 + torch.arange(c) % 16).cuda()
        flat[slots, r] = _scores(kind, c, 2 * c // 3, dtype)
        want[b] = flat[slots[2 * c // 3], :r]
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor(cl, dtype=torch.int32).cuda(), 0, SCALE[kind], 16, r)
    assert torch.equal(out[:, 0], want)


@pytest.mark.parametrize("kind", ["apart", "lagging"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [16, 32, 128])
def test_packed_rows_of_one_value(device, kind, dtype, heads):
    """Chunks of 128 rows, beside decodes where there are fewer heads."""
    gen = torch.Generator().manual_seed(3)
    r, ql, cl = 512, [40, 1, 1, 9], [900, 300, 1, 9]
    cache, tables = _pool(gen, cl, 16, r + 64, dtype)
    flat, q = cache[0].view(-1, r + 64), torch.zeros(sum(ql), heads, r + 64, dtype=dtype, device="cuda")
    q[..., r] = _factors(kind, heads, dtype)
    _values(kind, flat[:, :r])
    want, at = torch.zeros(sum(ql), heads, r, dtype=dtype, device="cuda"), 0
    for b, (n, c) in enumerate(zip(ql, cl)):
        slots = (tables[b, torch.arange(c) // 16].long() * 16 + torch.arange(c) % 16).cuda()
        flat[slots, r] = _scores(kind, c, c - n, dtype)
        want[at : at + n] = flat[slots[c - n], :r]  # seen by all of the sequence's queries
        at += n
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = latent_attention_varlen(q, cache, tables.cuda(), _cu(ql), ctx, 0, SCALE[kind], 16, max(ql), r)
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", ["apart", "lagging"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,ql,extra", [(128, [300, 213], [120, 87]), (112, [200, 120], [77, 300]), (3, [40, 2], [700, 9])])
def test_expanded_rows_of_one_value(device, kind, dtype, heads, ql, extra):
    """Eight, four and two waves a workgroup."""
    gen = torch.Generator().manual_seed(heads)
    cl = [a + b for a, b in zip(ql, extra)]
    q = torch.zeros(sum(ql), heads, 192, dtype=dtype, device="cuda")
    q[..., 128] = _factors(kind, heads, dtype)
    kv, kr = _randn(gen, sum(cl), heads, 256, dtype=dtype), torch.zeros(sum(cl), 64, dtype=dtype, device="cuda")
    _values(kind, kv[..., 128:])
    want, at, ck = torch.zeros(sum(ql), heads, 128, dtype=dtype, device="cuda"), 0, 0
    for n, c in zip(ql, cl):
        kr[ck : ck + c, 0] = _scores(kind, c, c - n, dtype)
        want[at : at + n] = kv[ck + c - n, :, 128:]
        at, ck = at + n, ck + c
    out = latent_attention_expanded(q, kv, kr, _cu(ql), _cu(cl), SCALE[kind], max(ql))
    assert torch.equal(out, want)


# Many keys far below one, whose values are large: a key with score 0 and value 1, n - 1 with score -25.5 (log2) and value
# 1024. The row is (1 + 1024 t) / (1 + t) with t = (n - 1) 2^-25.5. fp16 holds a probability of 2^-25.5 relative to the
# largest (which is taken as 2^7) to half of 2^-24 of it, 2^-6.5 of itself, which is that part of 1024 t; bf16, which has
# fp32's exponents, to 2^-8. The largest one's rounding is half a step of the type, fp32's are 2^-15 of the row at most, and
# the row's own is half a step: 2^-11 in fp16, and in bf16 (7 bits behind the first one: 2^-7 from 1 to the next value) 2^-8.
TAIL, LARGE = -25.5, 1024.0


def _check_tail(out: torch.Tensor, n: int) -> None:
    t = (n - 1) * 2.0**TAIL
    want = (1 + LARGE * t) / (1 + t)
    err = (out.double() - want).abs().max().item()
    half = torch.finfo(out.dtype).eps / 2
    assert err <= (2 * half + 2.0**-15) * want + 2.0**-6.5 * LARGE * t, (err, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,r,batch,n", [(16, 512, 700, 700), (32, 512, 600, 300), (64, 256, 600, 300), (128, 512, 520, 300)])
def test_many_keys_far_below_one(device, dtype, heads, r, batch, n):
    """More sequences than workgroups, so that the far keys stand beside the near one in a row's own sum."""
    blocks = -(-n // 16)
    cache = torch.zeros(1, blocks, 16, r + 64, dtype=dtype, device="cuda")
    flat = cache[0].view(-1, r + 64)
    flat[:, :r], flat[:, r] = LARGE, TAIL
    flat[0, :r], flat[0, r] = 1.0, 0.0
    q = torch.zeros(batch, heads, 1, r + 64, dtype=dtype, device="cuda")
    q[..., r] = 1.0
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").expand(batch, blocks)
    ctx = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    _check_tail(latent_attention_decode(q, cache, tables, ctx, 0, math.log(2), 16, r), n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,tq", [(128, 300), (112, 200), (3, 50)])
def test_many_keys_far_below_one_expanded(device, dtype, heads, tq):
    n = 700  # of which the last query sees all
    q = torch.zeros(tq, heads, 192, dtype=dtype, device="cuda")
    q[..., 128] = 1.0
    kv, kr = torch.zeros(n, heads, 256, dtype=dtype, device="cuda"), torch.zeros(n, 64, dtype=dtype, device="cuda")
    kv[..., 128:], kr[:, 0] = LARGE, TAIL
    kv[0, :, 128:], kr[0, 0] = 1.0, 0.0
    out = latent_attention_expanded(q, kv, kr, _cu([tq]), _cu([n]), math.log(2), tq)
    for j in (0, tq // 2, tq - 1):
        _check_tail(out[j], n - tq + j + 1)
