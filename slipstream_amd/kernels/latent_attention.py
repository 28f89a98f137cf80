"""Attention over latents on HIP, gfx950: keys and values of all heads from one latent a token.

With a head's projections ``W_k`` and ``W_v`` of the latent ``c`` and one rotated key ``r`` a token, the
score of a query ``[q_n | q_r]`` is ``q_n . W_k c + q_r . r`` and the output ``sum p W_v c``. Two forms:

* absorbed (``latent_attention_decode``, ``latent_attention_varlen``): the queries are ``[q_n W_k | q_r]``
  and the cached rows ``[c | r]`` are keys and (their latents) values, read from the pages once for all
  heads; ``W_v`` is applied to the output. For decodes and few new tokens.
* expanded (``latent_attention_expanded``): ``[W_k c | W_v c]`` is given for every token of the context; a
  third of the operations at the usual widths. For chunks of many tokens.

Names, arguments and rules are those of ``paged_attention_decode`` and ``paged_attention_varlen``: query j
of a sequence's ``n`` new tokens sees the keys ``[0, context - n + j]``, negative table entries are
masked, a row that sees no key gives zeros. The reference has no counterpart. bf16, fp16 and fp32;
latents (expanded: keys and values without their rotated part) up to 512 wide, rotated keys up to
256. A latent that a query does not see must be finite where one that it sees is in the same call's
new tokens. Device tensors only.

Scores, maxima and sums are fp32. Of bf16 and fp16 inputs the probabilities are rounded to the inputs' type
for the product with the values, and the sum that divides is of the rounded ones. Other widths than 256 or 512 and 64
(expanded: 128, 64 and 128), pages of fewer than eight tokens or no power of two of them, fp32, a scale of 0 and a cache
whose rows do not lie on 16 bytes run in a general kernel that is there for coverage.
"""

from __future__ import annotations

import torch

from slipstream_amd import _ffi
from slipstream_amd.kernels._common import launch, require_device, unit_last_stride
from slipstream_amd.kernels.latent_cache import check_latent_cache, layer_ptr
from slipstream_amd.kernels.paged_attention import _check_stream, _debug, _int32, _strides

_WS_BYTES: dict[tuple, int] = {}


def _workspace(device: torch.device, batch: int, tokens: int, tq: int, heads: int, latent_dim: int, rope_dim: int,
               dtype: int) -> torch.Tensor:
    """Scratch of this call alone, sized by the library: partial rows of keys split over workgroups."""
    key = (device.index, batch, tokens, tq, heads, latent_dim, rope_dim, dtype)
    nbytes = _WS_BYTES.get(key)
    if nbytes is None:
        need = _ffi.ctypes.c_int64(0)
        with torch.cuda.device(device):
            status = _ffi.lib().ss_latent_attention_workspace_size(batch, tokens, tq, heads, latent_dim, rope_dim,
                                                                   dtype, _ffi.ctypes.byref(need))
        _ffi.check(status, "latent attention workspace")
        if len(_WS_BYTES) > 4096:  # many distinct shapes: start over
            _WS_BYTES.clear()
        nbytes = _WS_BYTES[key] = max(int(need.value), 16)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _ints(x: torch.Tensor) -> torch.Tensor:
    """``x`` as a contiguous row of int32."""
    if x.dtype == torch.int32 and x.ndim == 1 and x.is_contiguous():
        return x
    return _int32(x.reshape(-1))


def _absorbed(who: str, q: torch.Tensor, out: torch.Tensor, latent_cache: torch.Tensor, block_tables: torch.Tensor,
              cu: torch.Tensor | None, ctx: torch.Tensor, layer_idx: int, scale: float, block_size: int,
              latent_dim: int, batch: int, tokens: int, tq: int, heads: int, q_strides, o_strides) -> torch.Tensor:
    if latent_cache.dtype != q.dtype:
        raise _ffi.KernelError(f"unsupported dtypes q={q.dtype} latent_cache={latent_cache.dtype} (must be equal)")
    dtype = _ffi.dtype_code(q.dtype)
    if latent_cache.stride(3) != 1:
        raise _ffi.KernelError(f"{who}: latent_cache must have a unit last stride")
    rope_dim = q.shape[-1] - latent_dim
    ws = _workspace(q.device, batch, tokens, tq, heads, latent_dim, rope_dim, dtype)
    if block_tables.dtype != torch.int32 or not block_tables.is_contiguous():
        block_tables = _int32(block_tables)
    ctx = _ints(ctx)
    cst = latent_cache.stride()
    page = cst[1] if latent_cache.shape[1] > 1 else block_size * cst[2]  # (of one page any will do)
    status = launch(
        q.device, _ffi.lib().ss_latent_attention, q.data_ptr(), out.data_ptr(), layer_ptr(latent_cache, layer_idx),
        block_tables.data_ptr(), None if cu is None else cu.data_ptr(), ctx.data_ptr(), batch, tokens, tq, heads,
        latent_dim, rope_dim, block_tables.shape[1], block_size, latent_cache.shape[1], _ffi.i64x3(*q_strides),
        _ffi.i64x3(*o_strides), _ffi.i64x2(page, cst[2]), block_tables.stride(0), float(scale), dtype,
        ws.data_ptr(), ws.numel())
    _ffi.check(status, who)
    return out


def _check_widths(q: torch.Tensor, latent_dim: int) -> None:
    if not 0 < latent_dim <= q.shape[-1]:
        raise ValueError(f"latent_dim {latent_dim} outside (0, {q.shape[-1]}], the width of q")


def latent_attention_decode(
    q: torch.Tensor,
    latent_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    layer_idx: int,
    scale: float,
    block_size: int,
    latent_dim: int,
) -> torch.Tensor:
    """The absorbed form for ``q [B, H, Tq, R + Dr]`` (the last Tq tokens of each sequence, typically one)
    over the paged latents of ``seq_lens[b]`` tokens; returns ``[B, Tq, H, R]`` in ``q``'s dtype, with
    ``R = latent_dim``. ``latent_cache [L, num_blocks, block_size, R + Dr]``."""
    if q.ndim != 4:
        raise ValueError(f"q must be [B, H, Tq, latent_dim + rope_dim], got {tuple(q.shape)}")
    batch, heads, tq, width = q.shape
    _check_widths(q, latent_dim)
    check_latent_cache(latent_cache, layer_idx, block_size, width)
    if block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be [B={batch}, max_blocks], got {tuple(block_tables.shape)}")
    if seq_lens.numel() != batch:
        raise ValueError(f"seq_lens has {seq_lens.numel()} entries for batch {batch}")
    out = q.new_empty((batch, tq, heads, latent_dim))
    if out.numel() == 0:
        return out
    require_device("latent_attention_decode", q, latent_cache, block_tables, seq_lens)
    q = unit_last_stride(q)
    so = out.stride()
    return _absorbed("latent_attention_decode", q, out, latent_cache, block_tables, None, seq_lens, layer_idx, scale,
                     block_size, latent_dim, batch, batch * tq, tq, heads, _strides(q, (0, 2, 1)), so[:3])


def latent_attention_varlen(
    q: torch.Tensor,
    latent_cache: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens: torch.Tensor,
    context_lens: torch.Tensor,
    layer_idx: int,
    scale: float,
    block_size: int,
    max_query_len: int,
    latent_dim: int,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The absorbed form for a packed step: ``q [T, H, R + Dr]`` holds every sequence's new tokens back to
    back, sequence ``b`` the tokens ``cu_seqlens[b]:cu_seqlens[b+1]`` and ``context_lens[b]`` cached ones
    (these tokens among them). Returns ``[T, H, R]`` (written into ``out`` when given: unit last
    stride); rows behind the last sequence are left as they are. A stream past ``T`` is clamped;
    ``max_query_len`` only tells how long sequences are likely to be (``SLIPSTREAM_DEBUG`` raises
    ``ValueError`` for a longer one and for a stream past ``T``)."""
    if q.ndim != 3:
        raise ValueError(f"q must be [T, H, latent_dim + rope_dim], got {tuple(q.shape)}")
    total, heads, width = q.shape
    _check_widths(q, latent_dim)
    check_latent_cache(latent_cache, layer_idx, block_size, width)
    batch = context_lens.numel()
    if cu_seqlens.numel() != batch + 1:
        raise ValueError(f"cu_seqlens must have batch+1={batch + 1} entries, got {cu_seqlens.numel()}")
    if block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError(f"block_tables must be [B={batch}, max_blocks], got {tuple(block_tables.shape)}")
    if max_query_len < 0:
        raise ValueError("max_query_len must be >= 0")
    if out is None:
        out = q.new_empty((total, heads, latent_dim))
    elif (out.shape != (total, heads, latent_dim) or out.dtype != q.dtype or out.device != q.device
          or out.stride(2) != 1):
        raise ValueError(f"out must be {(total, heads, latent_dim)} {q.dtype} on {q.device} with unit last stride")
    if batch == 0 or out.numel() == 0:
        return out
    require_device("latent_attention_varlen", q, latent_cache, block_tables, cu_seqlens, context_lens)
    q = unit_last_stride(q)
    cu = _ints(cu_seqlens)
    if _debug():
        _check_stream(cu, total, max_query_len)
    return _absorbed("latent_attention_varlen", q, out, latent_cache, block_tables, cu, context_lens, layer_idx, scale,
                     block_size, latent_dim, batch, total, max_query_len, heads, (0, *_strides(q, (0, 1))), (0, *_strides(out, (0, 1))))


def latent_attention_expanded(
    q: torch.Tensor,
    kv: torch.Tensor,
    k_rope: torch.Tensor,
    cu_seqlens: torch.Tensor,
    cu_context: torch.Tensor,
    scale: float,
    max_query_len: int,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The expanded form: ``q [T, H, Dn + Dr]`` as in ``latent_attention_varlen``; ``kv [S, H, Dn + Dv]`` the
    context's ``[W_k c | W_v c]`` and ``k_rope [S, Dr]`` its rotated keys, sequence ``b``'s in rows
    ``cu_context[b]:cu_context[b+1]``, its new tokens last. Returns ``[T, H, Dv]`` (written into ``out``
    when given: unit last stride); rows behind the last sequence are left as they are, and streams
    past ``T`` or ``S`` are clamped.

    The context's rows come from the cache by their slots: ``build_packed_step(block_tables,
    zeros, context_lens, ...)`` gives ``cu_context`` (its ``cu_seqlens``) and the slots, and
    ``rows = latent_cache[layer].view(-1, R + Dr).index_select(0, slots)`` the latents to project and,
    in ``rows[:, R:]``, ``k_rope``."""
    if q.ndim != 3 or kv.ndim != 3 or k_rope.ndim != 2:
        raise ValueError(f"q must be [T, H, Dn + Dr], kv [S, H, Dn + Dv] and k_rope [S, Dr]; got {tuple(q.shape)}, "
                         f"{tuple(kv.shape)} and {tuple(k_rope.shape)}")
    total, heads, width = q.shape
    keys, rope_dim = k_rope.shape
    nope = width - rope_dim
    value_dim = kv.shape[2] - nope
    if kv.shape[:2] != (keys, heads):
        raise ValueError(f"kv {tuple(kv.shape)} does not match k_rope's {keys} tokens and q's {heads} heads")
    if nope < 1 or value_dim < 1:
        raise ValueError(f"q is {width} wide, k_rope {rope_dim} and kv {kv.shape[2]}: no room for keys or values")
    batch = cu_seqlens.numel() - 1
    if batch < 0 or cu_context.numel() != batch + 1:
        raise ValueError(f"cu_seqlens and cu_context must have batch+1 entries, got {cu_seqlens.numel()} and "
                         f"{cu_context.numel()}")
    if max_query_len < 0:
        raise ValueError("max_query_len must be >= 0")
    if out is None:
        out = q.new_empty((total, heads, value_dim))
    elif (out.shape != (total, heads, value_dim) or out.dtype != q.dtype or out.device != q.device
          or out.stride(2) != 1):
        raise ValueError(f"out must be {(total, heads, value_dim)} {q.dtype} on {q.device} with unit last stride")
    if batch == 0 or out.numel() == 0:
        return out
    require_device("latent_attention_expanded", q, kv, k_rope, cu_seqlens, cu_context)
    if kv.dtype != q.dtype or k_rope.dtype != q.dtype:
        raise _ffi.KernelError(f"unsupported dtypes q={q.dtype} kv={kv.dtype} k_rope={k_rope.dtype} (must be equal)")
    dtype = _ffi.dtype_code(q.dtype)
    q, kv = unit_last_stride(q), unit_last_stride(kv)
    if rope_dim:
        k_rope = unit_last_stride(k_rope)
    cu, cu_ctx = _ints(cu_seqlens), _ints(cu_context)
    if _debug():
        _check_stream(cu, total, max_query_len)
        _check_stream(cu_ctx, keys, keys)
    # of one key any distance to the next will do: that of rows back to back, which every kernel takes
    ks = _strides(kv, (0, 1)) if keys > 1 else [heads * kv.shape[2], *_strides(kv, (1,))]
    status = launch(
        q.device, _ffi.lib().ss_latent_attention_expanded, q.data_ptr(), out.data_ptr(), kv.data_ptr(),
        k_rope.data_ptr(), cu.data_ptr(), cu_ctx.data_ptr(), batch, total, keys, max_query_len, heads, nope, rope_dim,
        value_dim, _ffi.i64x2(*_strides(q, (0, 1))), _ffi.i64x2(*_strides(out, (0, 1))), _ffi.i64x2(*ks),
        k_rope.stride(0) if keys > 1 else rope_dim, float(scale), dtype)
    _ffi.check(status, "latent_attention_expanded")
    return out
