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
    cos + cat(-x2, x1) * sin``. ``slot_mapping [N]``: slots below 0 or past the pool are skipped; a slot
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
    for c, name in ((cos, "cos"), (sin, "sin")):
        if c.shape != (n_tok, rope):
            raise ValueError(f"{name} {tuple(c.shape)} != [{n_tok}, {rope}]")
    if norm_weight is not None and norm_weight.shape != (width,):
        raise ValueError(f"norm_weight {tuple(norm_weight.shape)} != [{width}]")
    if slot_mapping.numel() != n_tok:
        raise ValueError(f"slot_mapping {slot_mapping.numel()} != tokens {n_tok}")
    check_latent_cache(latent_cache, layer_idx, block_size, width + rope)
    given = [q_rope, latent, k_rope, cos, sin, latent_cache] + ([] if norm_weight is None else [norm_weight])
    if any(t.dtype != q_rope.dtype for t in given):
        raise ValueError(f"all tensors must share one dtype, got {sorted({str(t.dtype) for t in given})}")
    dtype = _ffi.dtype_code(q_rope.dtype)
    if out is None:
        out = torch.empty((n_tok, heads, rope), dtype=q_rope.dtype, device=q_rope.device)
    elif out.shape != q_rope.shape or out.dtype != q_rope.dtype or out.device != q_rope.device:
        raise ValueError(f"out must be {tuple(q_rope.shape)} {q_rope.dtype} on {q_rope.device}")
    if n_tok == 0:
        return out
    require_device("latent_rope_and_cache", *given, slot_mapping)
    if any(t.shape[-1] > 1 and t.stride(-1) != 1 for t in (*given, out)):
        raise ValueError("every tensor needs a unit last stride")
    slots = slot_mapping.to(torch.int64).reshape(-1).contiguous()
    cst = latent_cache.stride()
    status = launch(
        q_rope.device, _ffi.lib().ss_latent_rope_and_cache, q_rope.data_ptr(), out.data_ptr(), latent.data_ptr(),
        k_rope.data_ptr(), cos.data_ptr(), sin.data_ptr(), None if norm_weight is None else norm_weight.data_ptr(),
        layer_ptr(latent_cache, layer_idx), slots.data_ptr(), n_tok, heads, width, rope, block_size,
        latent_cache.shape[1] * block_size, _ffi.i64x2(q_rope.stride(0), q_rope.stride(1)),
        _ffi.i64x2(out.stride(0), out.stride(1)), latent.stride(0), k_rope.stride(0), cos.stride(0), sin.stride(0),
        _ffi.i64x2(cst[1], cst[2]), eps, dtype)
    _ffi.check(status, "latent_rope_and_cache")
    return out
