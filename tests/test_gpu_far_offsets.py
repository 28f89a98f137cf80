"""e4m3 rows and product, the latent cache's write and expanded attention where elements lie more than 2^31 values and 2^32
bytes from a tensor's start: the same bits as from small tensors. (The absorbed form: test_gpu_latent.py.)"""

from __future__ import annotations

import pytest
import torch

from slipstream_amd.kernels import fp8_gemm, latent_attention_expanded, latent_rope_and_cache, quantize_fp8
from slipstream_amd.kernels.fp8_rows import FP8

pytestmark = pytest.mark.gpu


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


def test_rows(device):
    gen = torch.Generator().manual_seed(1)
    rows, cols = 170_003, 12_928  # 2.2e9 values
    last = _randn(gen, 5, cols)
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-5:] = last
    q, scale = quantize_fp8(x)
    want_q, want_scale = quantize_fp8(last)
    assert torch.equal(q[-5:].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(scale[-5:], want_scale)
    assert not scale[:-5].any() and not q[: rows // 2].view(torch.uint8).any()


def test_product(device):
    gen = torch.Generator().manual_seed(2)
    m, n, k = 80_003, 28_672, 128  # 2.3e9 results: of one block of keys, so that no split of them decides their order
    last = (torch.randn(3, k, generator=gen) * 50).to(FP8).cuda()
    w = (torch.randn(n, k, generator=gen) * 50).to(FP8).cuda()
    q = torch.zeros(m, k, dtype=torch.uint8, device="cuda").view(FP8)
    q.view(torch.uint8)[-3:] = last.view(torch.uint8)
    scale, ws = torch.ones(m, 1, device="cuda"), torch.full((n // 128, 1), 0.01, device="cuda")
    out = fp8_gemm(q, scale, w, ws)
    assert torch.equal(out[-3:], fp8_gemm(last, scale[-3:], w, ws)) and out[-3:].any() and not out[: m // 2].any()


def test_cache_write(device):
    gen = torch.Generator().manual_seed(3)
    r, d, bs, n = 512, 64, 64, 4
    blocks = (1 << 32) // (bs * (r + d) * 2) + 100
    cache = torch.zeros(1, blocks, bs, r + d, dtype=torch.bfloat16, device="cuda")
    small = torch.zeros(1, 1, bs, r + d, dtype=torch.bfloat16, device="cuda")
    q, rows, cs, sn, w = (_randn(gen, *s) for s in ((n, 2, d), (n, r + d), (n, d), (n, d), (r,)))
    args = (q, rows[:, :r], rows[:, r:], cs, sn)
    at = torch.tensor([bs - 1, 0, 5, 7], device="cuda")
    first = latent_rope_and_cache(*args, cache, (blocks - 1) * bs + at, 0, bs, w)
    second = latent_rope_and_cache(*args, small, at, 0, bs, w)
    assert torch.equal(first, second) and torch.equal(cache[0, -1], small[0, 0]) and small.any() and not cache[0, :-1].any()


@pytest.mark.parametrize("n", [520, 300, 4])  # eight, four and two waves a workgroup
def test_expanded(device, n):
    """Keys and values of the second sequence behind 2^32 bytes of the first one's."""
    gen = torch.Generator().manual_seed(4)
    heads, far = 128, 70_000
    q, kv, kr = _randn(gen, n, heads, 192), _randn(gen, 500, heads, 256), _randn(gen, 500, 64)
    all_kv = torch.zeros(far + 500, heads, 256, dtype=torch.bfloat16, device="cuda")
    all_kr = torch.zeros(far + 500, 64, dtype=torch.bfloat16, device="cuda")
    all_kv[far:], all_kr[far:] = kv, kr
    cu = torch.tensor([0, 0, n], dtype=torch.int32, device="cuda")
    out = latent_attention_expanded(q, all_kv, all_kr, cu, torch.tensor([0, far, far + 500], dtype=torch.int32, device="cuda"),
                                    0.1, n)
    want = latent_attention_expanded(q, kv, kr, cu[1:], torch.tensor([0, 500], dtype=torch.int32, device="cuda"), 0.1, n)
    assert torch.equal(out, want) and want.any()
