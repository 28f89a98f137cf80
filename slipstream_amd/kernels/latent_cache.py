"""The write of a paged cache of latents (HIP, gfx950): RMSNorm of a token's latent, rotary embedding
of its key and of the queries, and the scatter of ``[latent | key]``, in one launch.

What ``rope_and_cache`` is to a cache of keys and values, for layers whose heads share one latent a
token (``latent_attention_decode``). The cache is ``[num_layers, num_blocks, block_size, latent_dim +
rope_dim]`` (``slipstream_amd.paged_cache.allocate_latent_cache``), addressed by the same slots and
block tables. Everything is computed in fp32 and rounded once to the tensors' type. The reference has
no counterpart. Device tensors only.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device


def check_latent_cache(latent_cache: torch.Tensor, layer_idx: int, block_size: int, width: int) -> None:
    if latent_cache.ndim != 4:
        raise ValueError("latent_cache must be [num_layers, num_blocks, block_size, latent_dim + rope_dim]")
    if latent_cache.shape[2] != block_size:
        raise ValueError(f"latent_cache block_size {latent_cache.shape[2]} != block_size {block_size}")
    if latent_cache.shape[3] != width:
        raise ValueError(f"rows of latent_dim + rope_dim = {width} do not match the cache's {latent_cache.shape[3]}")
    if not 0 <= layer_idx < latent_cache.shape[0]:
        raise ValueError(f"layer_idx {layer_idx} out of range for {latent_cache.shape[0]} layers")


def layer_ptr(latent_cache: torch.Tensor, layer_idx: int) -> int:
    return latent_cache.data_ptr() + layer_idx * latent_cache.stride(0) * latent_cache.element_size()


def latent_rope_and_cache(
    q_rope: torch.Tensor,
    latent: torch.Tensor,
    k_rope: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    latent_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    layer_idx: int,
    block_size: int,
    norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Return ``rope(q_rope)`` and write ``[rms(latent) * norm_weight | rope(k_rope)]`` into
    ``latent_cache[layer_idx, slot // block_size, slot % block_size]``.

    ``q_rope [N, H, Dr]``, ``latent [N, R]``, ``k_rope [N, Dr]``, ``cos``/``sin [N, Dr]``, all with a unit
    last stride and any other (parts of the projections' outputs are taken as they are); ``rope(x) = x *
    cos + cat(-x2, x1) * sin`` with ``x = [x1, x2]``, as in ``rope_and_cache``: value ``i`` turns with value ``i + Dr / 2``.
    (Projections made for turning adjacent pairs need the rows of their rotated parts in the order ``0, 2, 4, .., 1, 3,
    5, ..``, of the queries in each head and of the key, once at load; scores stay the same.) ``slot_mapping [N]``: slots below 0 or past the pool are skipped; a slot
    that is given twice holds parts of either row. Without ``norm_weight [R]`` the latent is copied bit
    for bit. ``out`` (``[N, H, Dr]``, unit last stride, for instance the last columns of the absorbed
    queries; ``q_rope`` itself is allowed) takes the rotated queries.
    """
    if q_rope.ndim != 3 or latent.ndim != 2 or k_rope.ndim != 2:
        raise ValueError(f"q_rope must be [N, H, Dr], latent [N, R] and k_rope [N, Dr]; got {tuple(q_rope.shape)}, "
                         f"{tuple(latent.shape)} and {tuple(k_rope.shape)}")
    n_tok, heads, rope = q_rope.shape
    width = latent.shape[1]
    if rope % 2:
        raise ValueError(f"rope_dim must be even, got {rope}")
    if latent.shape[0] != n_tok or k_rope.shape != (n_tok, rope):
        raise ValueError(f"latent {tuple(latent.shape)} and k_rope {tuple(k_rope.shape)} do not match q_rope "
                         f"{tuple(q_rope.shape)}")
    if cos.shape != (n_tok, rope) or sin.shape != cos.shape:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be [{n_tok}, {rope}]")
    if norm_weight is not None and norm_weight.shape != (width,):
        raise ValueError(f"norm_weight {tuple(norm_weight.shape)} != [{width}]")
    if slot_mapping.numel() != n_tok:
        raise ValueError(f"slot_mapping {slot_mapping.numel()} != tokens {n_tok}")
    check_latent_cache(latent_cache, layer_idx, block_size, width + rope)
    weight = latent if norm_weight is None else norm_weight
    dtype, device = q_rope.dtype, q_rope.device
    if not dtype == latent.dtype == k_rope.dtype == cos.dtype == sin.dtype == latent_cache.dtype == weight.dtype:
        raise ValueError(f"all tensors must share one dtype, got {dtype}, {latent.dtype}, {k_rope.dtype}, {cos.dtype}, "
                         f"{sin.dtype}, {latent_cache.dtype} and {weight.dtype}")
    code = _ffi.dtype_code(dtype)
    if out is None:
        out = torch.empty((n_tok, heads, rope), dtype=dtype, device=device)
    elif out.shape != q_rope.shape or out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be {tuple(q_rope.shape)} {dtype} on {device}")
    if n_tok == 0:
        return out
    require_device("latent_rope_and_cache", q_rope, latent, k_rope, cos, sin, latent_cache, weight, slot_mapping)
    qs, os, ls, ks, cs, ss, cst = (q_rope.stride(), out.stride(), latent.stride(), k_rope.stride(), cos.stride(),
                                   sin.stride(), latent_cache.stride())
    # (of a tensor of one column any last stride will do)
    if (rope > 1 and not qs[2] == os[2] == ks[1] == cs[1] == ss[1] == 1) or cst[3] != 1 or (
            width > 1 and not ls[1] == weight.stride(-1) == 1):
        raise ValueError("every tensor needs a unit last stride")
    slots = slot_mapping
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    status = launch(
        device, _ffi.lib().ss_latent_rope_and_cache, q_rope.data_ptr(), out.data_ptr(), latent.data_ptr(),
        k_rope.data_ptr(), cos.data_ptr(), sin.data_ptr(), None if norm_weight is None else norm_weight.data_ptr(),
        layer_ptr(latent_cache, layer_idx), slots.data_ptr(), n_tok, heads, width, rope, block_size,
        latent_cache.shape[1] * block_size, _ffi.i64x2(qs[0], qs[1]), _ffi.i64x2(os[0], os[1]), ls[0], ks[0], cs[0],
        ss[0], _ffi.i64x2(cst[1], cst[2]), eps, code)
    _ffi.check(status, "latent_rope_and_cache")
    return out
