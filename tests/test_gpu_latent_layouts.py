"""Operands of other layouts than the usual: attention over latents from rows that do not lie on 16 bytes (the kernels that
the aligned ones take, bit for bit the same results), latents that the cache keeps as they are."""

from __future__ import annotations

import pytest
import torch
from test_gpu_latent import _pool, _randn

from slipstream_amd.kernels import (
    latent_attention_decode,
    latent_attention_expanded,
    latent_attention_varlen,
    latent_rope_and_cache,
)

pytestmark = pytest.mark.gpu


def _cu(n):
    return torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()


def _apart(x: torch.Tensor, before: int, behind: int) -> torch.Tensor:
    """``x`` as a part of rows that are ``before + behind`` values longer."""
    wide = torch.zeros((*x.shape[:-1], before + x.shape[-1] + behind), dtype=x.dtype, device=x.device)
    part = wide[..., before : before + x.shape[-1]]
    part.copy_(x)
    return part


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("before,behind", [(1, 0), (0, 1), (512, 3), (3, 5)])
def test_expanded_keys_of_any_alignment(device, dtype, before, behind):
    """The shared keys as the last columns of a projection that has an odd number of others; queries and the heads' keys
    likewise."""
    gen = torch.Generator().manual_seed(before + behind)
    heads, ql, cl = 4, [40, 3], [170, 90]
    q, kv = _randn(gen, sum(ql), heads, 192, dtype=dtype), _randn(gen, sum(cl), heads, 256, dtype=dtype)
    kr = _randn(gen, sum(cl), 64, dtype=dtype)
    args = (_cu(ql), _cu(cl), 0.1, max(ql))
    want = latent_attention_expanded(q, kv, kr, *args)
    assert torch.equal(latent_attention_expanded(q, kv, _apart(kr, before, behind), *args), want)
    got = latent_attention_expanded(_apart(q, before, behind), _apart(kv, before, behind), kr, *args)
    assert torch.equal(got, want)


def _odd(x: torch.Tensor) -> torch.Tensor:
    """Strides of the dimensions of size one that are no multiple of anything."""
    return x.as_strided(x.shape, [s if n > 1 or i == x.ndim - 1 else 7 for i, (s, n) in enumerate(zip(x.stride(), x.shape))])


@pytest.mark.parametrize("heads,tokens,keys", [(1, 5, 9), (4, 1, 1), (1, 1, 1), (1, 1, 40)])
def test_expanded_of_one_head_or_token(device, heads, tokens, keys):
    """A stride that no second head or token uses may be anything."""
    gen = torch.Generator().manual_seed(heads + keys)
    q, kv, kr = (_randn(gen, *s, dtype=torch.bfloat16) for s in ((tokens, heads, 192), (keys, heads, 256), (keys, 64)))
    args = (_cu([tokens]), _cu([keys]), 0.1, tokens)
    want = latent_attention_expanded(q, kv, kr, *args)

    assert torch.equal(latent_attention_expanded(_odd(q), _odd(kv), _odd(kr), *args), want)


@pytest.mark.parametrize("heads", [1, 16, 128])
def test_absorbed_of_one_page_or_sequence(device, heads):
    gen = torch.Generator().manual_seed(heads)
    cache, tables = _randn(gen, 1, 1, 16, 576, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    q, ctx = _randn(gen, 1, heads, 1, 576, dtype=torch.bfloat16), torch.tensor([13], dtype=torch.int32, device="cuda")
    want = latent_attention_decode(q, cache, tables, ctx, 0, 0.05, 16, 512)
    assert torch.equal(latent_attention_decode(_odd(q), _odd(cache), _odd(tables), ctx, 0, 0.05, 16, 512), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,r,ql,extra", [(16, 512, [1, 1, 1], [30, 700, 0]), (64, 256, [1, 3], [90, 400]),
                                              (128, 512, [2, 1], [300, 2000]), (16, 512, [40, 1], [500, 30])])
def test_absorbed_outputs_of_any_alignment(device, dtype, heads, r, ql, extra):
    """Rows of ``out`` that begin at any value, whole items and merged ones; what lies beside them stays."""
    gen = torch.Generator().manual_seed(heads)
    cl = [a + b for a, b in zip(ql, extra)]
    cache, tables = _pool(gen, cl, 16, r + 64, dtype)
    q = _randn(gen, sum(ql), heads, r + 64, dtype=dtype)
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    args = (tables.cuda(), _cu(ql), ctx, 0, 0.06, 16, max(ql), r)
    want = latent_attention_varlen(q, cache, *args)
    for before in (1, 2, 3):
        wide = torch.full((sum(ql), heads, r + 4), 9.0, dtype=dtype, device="cuda")
        got = latent_attention_varlen(q, cache, *args, out=wide[..., before : before + r])
        assert torch.equal(got, want)
        assert (wide[..., :before] == 9).all() and (wide[..., before + r :] == 9).all()
        wide = torch.full((sum(ql), heads * r + 5), 9.0, dtype=dtype, device="cuda")
        part = wide[:, before : before + heads * r].unflatten(1, (heads, r))
        assert torch.equal(latent_attention_varlen(q, cache, *args, out=part), want)
        assert (wide[:, :before] == 9).all() and (wide[:, before + heads * r :] == 9).all()


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, torch.int16), (torch.float16, torch.int16), (torch.float32, torch.int32)])
@pytest.mark.parametrize("before", [0, 1])
def test_latents_without_a_norm_keep_every_bit(device, dtype, bits, before):
    """Every 16-bit pattern, NaN that signal and subnormals among them (fp32: each with 16 other bits behind it)."""
    n, r, d = 128, 512, 8
    codes = torch.arange(1 << 16, dtype=torch.int32, device="cuda")
    codes = (codes << 16 | (codes * 40503 & 0xFFFF)) if bits == torch.int32 else (codes - 32768).to(bits)
    latent = _apart(codes.view(n, r), before, 0)  # 16 bytes a piece, or a value
    ones = torch.ones(n, 1, d, dtype=dtype, device="cuda")
    cache = torch.zeros(1, n // 16, 16, r + d, dtype=dtype, device="cuda")
    latent_rope_and_cache(ones, latent.view(dtype), ones[:, 0], ones[:, 0], ones[:, 0], cache, torch.arange(n, device="cuda"), 0, 16)
    assert torch.equal(cache.view(bits).view(n, r + d)[:, :r], codes.view(n, r))
