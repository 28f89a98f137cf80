"""Packed steps of the absorbed form whose one-token sequences and others go in two launches, each with its part of the
workspace and its merge, and tiles of 16, 32 and 64 rows of several tokens; against the float64 oracle."""

from __future__ import annotations

import pytest
import torch
from test_gpu_latent import _check_absorbed, _pool, _randn

from slipstream_amd.kernels import latent_attention_varlen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r", [512, 256])
@pytest.mark.parametrize("heads,ql,extra,longest", [
    (64, [1, 1, 70, 1, 9], [300, 2500, 900, 0, 40], 70),  # 64 rows beside 128
    (40, [1, 9, 1, 40], [3000, 0, 33, 1200], 40),
    (33, [1, 1, 5], [64, 700, 100], 5),
    (16, [1, 4, 2, 1], [2600, 800, 31, 5], 4),  # 16 beside 64
    (16, [1, 2, 0, 2, 1], [40, 1900, 7, 0, 900], 2),  # 16 beside 32
    (8, [1, 4, 3], [1500, 2200, 0], 4),  # 16 beside 32, four tokens an item
    (5, [3, 1, 12, 1], [100, 3000, 2000, 1], 12),  # 16 beside 64, twelve tokens
    (20, [1, 3, 2], [700, 0, 3000], 3),  # 32 beside 64
    (2, [8, 8, 8], [0, 1000, 77], 8),  # 16 alone, eight tokens an item
    (4, [8, 8], [3000, 12], 8),  # 32 alone
    (6, [10, 10, 10], [2000, 9, 300], 10),  # 64 alone
])
def test_steps_of_few_rows_beside_more(device, dtype, r, heads, ql, extra, longest):
    gen = torch.Generator().manual_seed(heads + r)
    cl = [a + b for a, b in zip(ql, extra)]
    cache, tables = _pool(gen, cl, 16, r + 64, dtype)
    total = sum(ql)
    q = _randn(gen, total + 2, heads, r + 64, dtype=dtype)
    cu = torch.tensor([0] + ql).cumsum(0).to(torch.int32).cuda()
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = torch.full((total + 2, heads, r), 5.0, dtype=dtype, device="cuda")

    def step():
        return latent_attention_varlen(q, cache, tables.cuda(), cu, ctx, 0, 0.06, 16, longest, r, out=out)

    step()
    _check_absorbed(out, q, cache[0], tables, ql, cl, 0.06, r, dtype)
    assert (out[total:] == 5).all()
    first = out.clone()
    for _ in range(3):
        out.fill_(5.0)
        assert torch.equal(step(), first)


@pytest.mark.parametrize("heads,ql,longest", [(64, [1, 1, 20, 1], 20), (16, [1, 3, 1, 2], 4)])
def test_two_launches_in_a_graph(device, heads, ql, longest):
    """Replayed with other lengths: sequences of one token become longer ones and the other way round."""
    gen = torch.Generator().manual_seed(heads)
    cache, tables = _pool(gen, [900] * len(ql), 16, 576, torch.bfloat16)
    tables, total = tables.cuda(), sum(ql)
    q = _randn(gen, total, heads, 576, dtype=torch.bfloat16)
    cu = torch.tensor([0] + ql).cumsum(0).to(torch.int32).cuda()
    ctx = torch.tensor([700, 40, 300, 90], dtype=torch.int32).cuda()

    def step():
        return latent_attention_varlen(q, cache, tables, cu, ctx, 0, 0.06, 16, longest, 512)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        lens = ql[turn:] + ql[:turn]
        cu.copy_(torch.tensor([0] + lens).cumsum(0))
        ctx.copy_(torch.tensor([700 - 100 * turn, 40 + 3 * turn, 300, 90 + 200 * turn]))
        q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, step())
        _check_absorbed(held, q, cache[0], tables.cpu(), lens, ctx.tolist(), 0.06, 512, torch.bfloat16)
