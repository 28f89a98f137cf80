"""Attention over latents on the GPU at the sizes that decide between its kernels, their splits and their
merges, and in graphs and on streams that run at once; against the float64 oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from test_gpu_latent import _check_absorbed, _check_expanded, _pool, _randn

from slipstream_amd.kernels import fp8_gemm, latent_attention_decode, latent_attention_expanded, latent_attention_varlen

pytestmark = pytest.mark.gpu


def _cu(n):
    return torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,ql,extra", [
    (128, [300, 7, 213, 1], [120, 0, 87, 400]),  # eight waves a workgroup
    (112, [200, 1, 120], [77, 300, 0]),  # four
    (17, [3, 1, 40, 2], [5, 600, 129, 0]),  # two, heads that are no multiple of the XCDs
])
def test_expanded_workgroups(device, dtype, heads, ql, extra):
    gen = torch.Generator().manual_seed(heads)
    cl = [a + b for a, b in zip(ql, extra)]
    q, kv = _randn(gen, sum(ql), heads, 192, dtype=dtype), _randn(gen, sum(cl), heads, 256, dtype=dtype)
    kr = _randn(gen, sum(cl), 64, dtype=dtype)
    out = latent_attention_expanded(q, kv, kr, _cu(ql), _cu(cl), 0.1, max(ql))
    _check_expanded(out, q, kv, kr, ql, cl, 0.1, 128, dtype)
    assert torch.equal(latent_attention_expanded(q, kv, kr, _cu(ql), _cu(cl), 0.1, max(ql)), out)


def test_expanded_many_sequences(device):
    """More sequences than are ordered at once, some without tokens, some of equal length."""
    rng = np.random.default_rng(5)
    ql = [int(n) for n in rng.integers(0, 9, 150)]
    cl = [n + int(e) for n, e in zip(ql, rng.integers(0, 90, 150))]
    gen = torch.Generator().manual_seed(6)
    q, kv = _randn(gen, sum(ql), 9, 192, dtype=torch.bfloat16), _randn(gen, sum(cl), 9, 256, dtype=torch.bfloat16)
    kr = _randn(gen, sum(cl), 64, dtype=torch.bfloat16)
    out = latent_attention_expanded(q, kv, kr, _cu(ql), _cu(cl), 0.1, max(ql))
    _check_expanded(out, q, kv, kr, ql, cl, 0.1, 128, torch.bfloat16)


@pytest.mark.parametrize("heads,batch,most", [(16, 700, 90), (32, 300, 90), (64, 600, 60), (128, 300, 200)])
def test_decode_many_sequences(device, heads, batch, most):
    """More sequences than a workgroup has threads, with empty ones among them and runs of short ones."""
    rng = np.random.default_rng(heads)
    cl = [int(n) for n in rng.integers(0, most, batch)]
    cl[3:40] = [0] * 37
    cl[60:120] = [1] * 60
    gen = torch.Generator().manual_seed(heads)
    cache, tables = _pool(gen, cl, 16, 576, torch.bfloat16)
    q = _randn(gen, batch, heads, 1, 576, dtype=torch.bfloat16)
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor(cl, dtype=torch.int32).cuda(), 0, 0.06, 16, 512)
    _check_absorbed(out[:, 0], q[:, :, 0], cache[0], tables, [1] * batch, cl, 0.06, 512, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,r,cl", [(16, 512, [7000]), (128, 512, [6000]), (128, 256, [2500, 3, 1800]),
                                        (64, 512, [3000, 0, 1]), (33, 512, [1, 4000]), (16, 256, [900] * 12)])
def test_few_long_contexts(device, dtype, heads, r, cl):
    """Keys split over many workgroups and joined: right, the same each time, and whatever the batch is padded with."""
    gen = torch.Generator().manual_seed(heads + len(cl))
    cache, tables = _pool(gen, cl, 64, r + 64, dtype)
    q = _randn(gen, len(cl), heads, 1, r + 64, dtype=dtype)
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = latent_attention_decode(q, cache, tables.cuda(), ctx, 0, 0.06, 64, r)
    _check_absorbed(out[:, 0], q[:, :, 0], cache[0], tables, [1] * len(cl), cl, 0.06, r, dtype)
    for _ in range(3):
        assert torch.equal(latent_attention_decode(q, cache, tables.cuda(), ctx, 0, 0.06, 64, r), out)


@pytest.mark.parametrize("heads,ql,extra", [(128, [150, 1, 1, 33, 0, 1], [500, 900, 30, 0, 10, 1]),
                                            (16, [300, 1, 1, 9, 260], [900, 2000, 3, 70, 0]),
                                            (160, [20, 1, 3], [90, 400, 33]), (300, [2, 1], [100, 5])])
def test_mixed_steps(device, heads, ql, extra):
    """Chunks of many items beside decodes; more heads than a workgroup has rows."""
    gen = torch.Generator().manual_seed(heads)
    cl = [a + b for a, b in zip(ql, extra)]
    cache, tables = _pool(gen, cl, 16, 576, torch.bfloat16)
    q = _randn(gen, sum(ql), heads, 576, dtype=torch.bfloat16)
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = latent_attention_varlen(q, cache, tables.cuda(), _cu(ql), ctx, 0, 0.06, 16, max(ql), 512)
    _check_absorbed(out, q, cache[0], tables, ql, cl, 0.06, 512, torch.bfloat16)


def test_graphs_and_streams_at_once(device):
    """Two graphs and an eager call on three streams, several times over with other lengths: every result is
    the eager one's."""
    gen = torch.Generator().manual_seed(2)
    work = []
    for heads, cl in ((16, [400, 30]), (128, [900, 5, 70])):
        cache, tables = _pool(gen, cl, 16, 576, torch.bfloat16)
        q = _randn(gen, len(cl), heads, 1, 576, dtype=torch.bfloat16)
        work.append((q, cache, tables.cuda(), torch.tensor(cl, dtype=torch.int32).cuda()))
    x = torch.randint(0, 120, (300, 2048), generator=gen).to(torch.uint8).cuda().view(torch.float8_e4m3fn)
    w = torch.randint(0, 120, (512, 2048), generator=gen).to(torch.uint8).cuda().view(torch.float8_e4m3fn)
    sx, sw = torch.rand(300, 16, generator=gen).cuda(), torch.rand(4, 16, generator=gen).cuda()

    def run(i):
        q, cache, tables, ctx = work[i]
        return latent_attention_decode(q, cache, tables, ctx, 0, 0.06, 16, 512), fp8_gemm(x, sx, w, sw)

    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    for i in range(2):
        run(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            held = run(i)
        graphs.append((graph, held))
    for turn in range(4):
        for q, _, _, ctx in work:
            ctx.sub_(turn)
            q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        sx.mul_(1.5)
        want = [run(0), run(1)]
        torch.cuda.synchronize()
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        with torch.cuda.stream(streams[2]):
            got.append(run(turn % 2))
        torch.cuda.synchronize()
        got += [held for _, held in graphs]
        for have, need in zip(got, (want[turn % 2], want[0], want[1])):
            assert torch.equal(have[0], need[0]) and torch.equal(have[1], need[1])


@pytest.mark.parametrize("heads", [2, 16, 32])
@pytest.mark.parametrize("ql,extra", [([1, 1, 1], [300, 0, 2000]), ([5, 40], [100, 7]), ([0, 1, 0, 9], [4, 90, 0, 700]),
                                      ([0, 0, 0], [5, 0, 9])])
def test_steps_of_one_kind(device, heads, ql, extra):
    """Decodes alone, chunks alone or nothing at all in a call that may hold both."""
    gen = torch.Generator().manual_seed(heads + len(ql))
    cl = [a + b for a, b in zip(ql, extra)]
    cache, tables = _pool(gen, cl, 16, 576, torch.bfloat16)
    q = _randn(gen, sum(ql) + 1, heads, 576, dtype=torch.bfloat16)
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = torch.full((sum(ql) + 1, heads, 512), 5.0, dtype=torch.bfloat16, device="cuda")
    latent_attention_varlen(q, cache, tables.cuda(), _cu(ql), ctx, 0, 0.06, 16, 64, 512, out=out)
    _check_absorbed(out, q, cache[0], tables, ql, cl, 0.06, 512, torch.bfloat16)
    assert (out[sum(ql) :] == 5).all()


@pytest.mark.parametrize("heads", [16, 64, 128])
@pytest.mark.parametrize("bs", [8, 256, 2048])
def test_page_sizes(device, heads, bs):
    """Pages of fewer keys than a tile and of many tiles, and one that is shared by two sequences."""
    cl = [70, 9, 2100, 8]
    gen = torch.Generator().manual_seed(heads + bs)
    cache, tables = _pool(gen, cl, bs, 576, torch.float16)
    tables[1, 0] = tables[0, 0]
    q = _randn(gen, len(cl), heads, 1, 576, dtype=torch.float16)
    out = latent_attention_decode(q, cache, tables.cuda(), torch.tensor(cl, dtype=torch.int32).cuda(), 0, 0.06, bs, 512)
    _check_absorbed(out[:, 0], q[:, :, 0], cache[0], tables, [1] * len(cl), cl, 0.06, 512, torch.float16)


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_scores_that_overflow_and_hold_nan(device, heads):
    """A latent with a NaN makes the rows that see it NaN, one with an infinity not finite, and no others; of scores far
    apart the largest one's values are left."""
    gen = torch.Generator().manual_seed(heads)
    cl = [100, 300, 40, 90]
    cache, tables = _pool(gen, cl, 16, 576, torch.bfloat16)
    cache[0, tables[1, 7].item(), 3, 5] = float("nan")
    cache[0, tables[2, 1].item(), 2, 9] = float("inf")
    q = _randn(gen, 4, heads, 1, 576, dtype=torch.bfloat16)
    ctx = torch.tensor(cl, dtype=torch.int32).cuda()
    out = latent_attention_decode(q, cache, tables.cuda(), ctx, 0, 0.06, 16, 512)[:, 0]
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0].float()).all() and torch.isfinite(out[3].float()).all()
    assert not torch.isfinite(out[2].float()).all()
    good = [0, 3]
    _check_absorbed(out[good], q[good, :, 0], cache[0], tables[good], [1, 1], [100, 90], 0.06, 512, torch.bfloat16)
    sharp = latent_attention_decode(q[:1], cache, tables[:1].cuda(), ctx[:1], 0, 3000.0, 16, 512)[:, 0]
    rows = cache[0][tables[0, :7].long().cuda()].reshape(-1, 576)[:100].float()
    best = (q[0, :, 0].float() @ rows.t()).argmax(dim=1)
    # all but the best row's probabilities are 2^-1000 and less of it. Its own is 2^(score - m) for the maximum m that was
    # last taken (up to 2^8), rounded to bf16 for the product but not in the sum that divides: half a step (2^-8) of the
    # value, and another when the output is rounded, 2^-7 + 2^-16 together
    want = rows[best, :512]
    assert ((sharp[0].float() - want).abs() <= (2.0**-7 + 2.0**-15) * want.abs()).all()
