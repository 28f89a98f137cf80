"""Attention over latents and the latent cache's write: host checks (shapes, dtypes, devices, the C ABI's
own), and the oracle against known answers (no GPU needed)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import latent as ora
from slipstream_amd import _ffi
from slipstream_amd.kernels import (
    latent_attention_decode,
    latent_attention_expanded,
    latent_attention_varlen,
    latent_rope_and_cache,
)
from slipstream_amd.paged_cache import allocate_latent_cache

FAKE = 1 << 20  # a 16-byte aligned address that no refused call reads
CACHE = allocate_latent_cache(2, 5, 16, 32, 8, dtype=torch.bfloat16, device=torch.device("cpu"))


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _write(**change):
    a = {"q_rope": _bf(6, 3, 8), "latent": _bf(6, 32), "k_rope": _bf(6, 8), "cos": _bf(6, 8), "sin": _bf(6, 8),
         "latent_cache": CACHE, "slot_mapping": torch.arange(6), "layer_idx": 1, "block_size": 16,
         "norm_weight": _bf(32)}
    return latent_rope_and_cache(**{**a, **change})


def _decode(**change):
    a = {"q": _bf(2, 3, 1, 40), "latent_cache": CACHE, "block_tables": torch.zeros(2, 4, dtype=torch.int32),
         "seq_lens": torch.ones(2, dtype=torch.int32), "layer_idx": 1, "scale": 1.0, "block_size": 16, "latent_dim": 32}
    return latent_attention_decode(**{**a, **change})


def _varlen(**change):
    a = {"q": _bf(6, 3, 40), "latent_cache": CACHE, "block_tables": torch.zeros(2, 4, dtype=torch.int32),
         "cu_seqlens": torch.tensor([0, 2, 6], dtype=torch.int32), "context_lens": torch.tensor([9, 9], dtype=torch.int32),
         "layer_idx": 1, "scale": 1.0, "block_size": 16, "max_query_len": 4, "latent_dim": 32}
    return latent_attention_varlen(**{**a, **change})


def _expanded(**change):
    a = {"q": _bf(6, 3, 24), "kv": _bf(20, 3, 32), "k_rope": _bf(20, 8), "scale": 1.0, "max_query_len": 4,
         "cu_seqlens": torch.tensor([0, 2, 6], dtype=torch.int32), "cu_context": torch.tensor([0, 9, 20], dtype=torch.int32)}
    return latent_attention_expanded(**{**a, **change})


@pytest.mark.parametrize("call,change,match", [
    (_write, {"q_rope": _bf(6, 24)}, "q_rope"),
    (_write, {"q_rope": _bf(6, 3, 7)}, "even"),
    (_write, {"latent": _bf(5, 32)}, "do not match"),
    (_write, {"k_rope": _bf(6, 6)}, "do not match"),
    (_write, {"cos": _bf(1, 8)}, "cos"),
    (_write, {"sin": _bf(6, 4)}, "sin"),
    (_write, {"norm_weight": _bf(31)}, "norm_weight"),
    (_write, {"slot_mapping": torch.arange(5)}, "slot_mapping"),
    (_write, {"layer_idx": 2}, "out of range"),
    (_write, {"layer_idx": -1}, "out of range"),
    (_write, {"block_size": 8}, "block_size"),
    (_write, {"latent": _bf(6, 31), "norm_weight": None}, "match"),
    (_write, {"latent_cache": CACHE[0]}, "num_layers"),
    (_write, {"cos": torch.zeros(6, 8)}, "share one dtype"),
    (_write, {"out": _bf(6, 3, 4)}, "out must be"),
    (_decode, {"q": _bf(2, 3, 40)}, "q must be"),
    (_decode, {"latent_dim": 0}, "latent_dim"),
    (_decode, {"latent_dim": 41}, "latent_dim"),
    (_decode, {"q": _bf(2, 3, 1, 41)}, "do not match"),
    (_decode, {"block_size": 32}, "block_size"),
    (_decode, {"layer_idx": 2}, "out of range"),
    (_decode, {"block_tables": torch.zeros(3, 4, dtype=torch.int32)}, "block_tables"),
    (_decode, {"seq_lens": torch.ones(3, dtype=torch.int32)}, "seq_lens"),
    (_varlen, {"q": _bf(2, 3, 1, 40)}, "q must be"),
    (_varlen, {"latent_dim": -3}, "latent_dim"),
    (_varlen, {"cu_seqlens": torch.zeros(2, dtype=torch.int32)}, "cu_seqlens"),
    (_varlen, {"block_tables": torch.zeros(4, dtype=torch.int32)}, "block_tables"),
    (_varlen, {"max_query_len": -1}, "max_query_len"),
    (_varlen, {"out": _bf(6, 3, 40)}, "out must be"),
    (_varlen, {"out": torch.zeros(6, 3, 32)}, "out must be"),
    (_expanded, {"q": _bf(6, 24)}, "q must be"),
    (_expanded, {"kv": _bf(20, 2, 32)}, "does not match"),
    (_expanded, {"k_rope": _bf(19, 8)}, "does not match"),
    (_expanded, {"k_rope": _bf(20, 24)}, "no room"),
    (_expanded, {"kv": _bf(20, 3, 16)}, "no room"),
    (_expanded, {"cu_context": torch.zeros(2, dtype=torch.int32)}, "cu_context"),
    (_expanded, {"max_query_len": -1}, "max_query_len"),
    (_expanded, {"out": _bf(6, 3, 24)}, "out must be"),
])
def test_shapes_and_types_are_refused(call, change, match):
    with pytest.raises(ValueError, match=match):
        call(**change)


@pytest.mark.parametrize("call", [_write, _decode, _varlen, _expanded])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="HIP devices only"):
        call()


def test_empty_calls_compute_nothing():
    none = {"latent": _bf(0, 32), "k_rope": _bf(0, 8), "cos": _bf(0, 8), "sin": _bf(0, 8), "slot_mapping": torch.arange(0)}
    assert _write(q_rope=_bf(0, 3, 8), **none).shape == (0, 3, 8)
    no_seqs = {"block_tables": torch.zeros(0, 4, dtype=torch.int32)}
    assert _decode(q=_bf(0, 3, 1, 40), seq_lens=torch.ones(0), **no_seqs).shape == (0, 1, 3, 32)
    assert _decode(q=_bf(2, 0, 1, 40)).shape == (2, 1, 0, 32)
    assert _varlen(q=_bf(0, 3, 40)).shape == (0, 3, 32)
    assert _expanded(q=_bf(0, 3, 24)).shape == (0, 3, 16)


def test_c_entries_refuse_before_any_launch():
    lib = _ffi.lib()
    two, three = _ffi.i64x2(0, 0), _ffi.i64x3(0, 0, 0)

    def absorbed(batch=1, total=1, tq=1, heads=2, r=512, d=64, bs=16, dtype=1, q=FAKE, cu=None, width=4, pool=4):
        return lib.ss_latent_attention(q, FAKE, FAKE, FAKE, cu, FAKE, batch, total, tq, heads, r, d, width, bs, pool, three,
                                       three, two, 4, 1.0, dtype, None, 0, None)

    assert absorbed(batch=-1) == _ffi.SS_ERR_INVALID and absorbed(heads=-1) == _ffi.SS_ERR_INVALID
    assert absorbed(tq=-1) == _ffi.SS_ERR_INVALID and absorbed(cu=FAKE, total=-1) == _ffi.SS_ERR_INVALID
    assert absorbed(bs=0) == _ffi.SS_ERR_INVALID and absorbed(width=-1) == _ffi.SS_ERR_INVALID
    assert absorbed(q=None) == _ffi.SS_ERR_INVALID and b"null" in lib.ss_last_error()
    assert absorbed(dtype=7) == _ffi.SS_ERR_UNSUPPORTED
    for r, d in ((513, 64), (0, 64), (512, 257), (512, -1)):
        assert absorbed(r=r, d=d) == _ffi.SS_ERR_UNSUPPORTED, (r, d)
    assert absorbed(batch=1 << 21) == _ffi.SS_ERR_UNSUPPORTED
    assert absorbed(batch=0, q=None) == _ffi.SS_OK and absorbed(heads=0, q=None) == _ffi.SS_OK
    assert absorbed(tq=0, q=None) == _ffi.SS_OK and absorbed(cu=FAKE, total=0, q=None) == _ffi.SS_OK
    need = ctypes.c_int64(-1)
    size = lib.ss_latent_attention_workspace_size
    assert size(1, 1, 1, 16, 512, 64, 1, None) == _ffi.SS_ERR_INVALID
    assert size(1, 1, 1, 16, 513, 64, 1, ctypes.byref(need)) == _ffi.SS_ERR_UNSUPPORTED
    assert size(-1, 1, 1, 16, 512, 64, 1, ctypes.byref(need)) == _ffi.SS_ERR_INVALID

    def expanded(batch=1, total=1, keys=1, heads=2, n=128, d=64, v=128, dtype=1, kv=FAKE, rope=FAKE):
        return lib.ss_latent_attention_expanded(FAKE, FAKE, kv, rope, FAKE, FAKE, batch, total, keys, 1, heads, n, d, v, two,
                                                two, two, 0, 1.0, dtype, None)

    assert expanded(batch=-1) == _ffi.SS_ERR_INVALID and expanded(keys=-1) == _ffi.SS_ERR_INVALID
    assert expanded(kv=None) == _ffi.SS_ERR_INVALID and expanded(rope=None) == _ffi.SS_ERR_INVALID
    assert expanded(dtype=7) == _ffi.SS_ERR_UNSUPPORTED and expanded(v=513) == _ffi.SS_ERR_UNSUPPORTED
    assert expanded(n=0) == _ffi.SS_ERR_UNSUPPORTED and expanded(d=257) == _ffi.SS_ERR_UNSUPPORTED
    assert expanded(batch=0, kv=None) == _ffi.SS_OK

    def write(n=1, heads=2, r=512, d=64, bs=16, dtype=1, latent=FAKE, q=FAKE, rope=FAKE):
        return lib.ss_latent_rope_and_cache(q, FAKE, latent, rope, FAKE, FAKE, None, FAKE, FAKE, n, heads, r, d, bs, 64, two,
                                            two, 0, 0, 0, 0, two, 1e-6, dtype, None)

    assert write(n=-1) == _ffi.SS_ERR_INVALID and write(d=63) == _ffi.SS_ERR_INVALID and write(bs=0) == _ffi.SS_ERR_INVALID
    assert write(latent=None) == _ffi.SS_ERR_INVALID and write(q=None) == _ffi.SS_ERR_INVALID
    assert write(rope=None) == _ffi.SS_ERR_INVALID
    assert write(dtype=7) == _ffi.SS_ERR_UNSUPPORTED and write(n=1 << 24) == _ffi.SS_ERR_UNSUPPORTED
    assert write(n=0, latent=None) == _ffi.SS_OK


def test_oracle_is_the_heads_own_attention():
    """The absorbed form equals attention with keys W_k c and values W_v c of each head, and torch's own
    attention in float64; the expanded form's arguments give the same."""
    rng = np.random.default_rng(0)
    heads, r, dn, dr, dv, n, s = 3, 16, 8, 4, 6, 3, 11
    c, kr = rng.normal(size=(s, r)), rng.normal(size=(s, dr))
    wk, wv = rng.normal(size=(heads, dn, r)), rng.normal(size=(heads, dv, r))
    qn, qr = rng.normal(size=(n, heads, dn)), rng.normal(size=(n, heads, dr))
    valid = np.ones(s, dtype=bool)
    absorbed, _, _ = ora.attend(np.concatenate([np.einsum("nhd,hdr->nhr", qn, wk), qr], -1), np.concatenate([c, kr], -1), c,
                                valid, s, 0.3)
    k, v = np.einsum("sr,hdr->shd", c, wk), np.einsum("sr,hdr->shd", c, wv)
    full = np.concatenate([k, np.repeat(kr[:, None], heads, 1)], -1)
    expanded, _, _ = ora.attend(np.concatenate([qn, qr], -1), full, v, valid, s, 0.3)
    assert np.allclose(np.einsum("nhr,hdr->nhd", absorbed, wv), expanded, atol=1e-12)
    mask = torch.ones(n, s, dtype=torch.bool).tril(s - n)
    sdpa = torch.nn.functional.scaled_dot_product_attention(
        *(torch.from_numpy(a).transpose(0, 1) for a in (np.concatenate([qn, qr], -1), full, v)), attn_mask=mask, scale=0.3)
    assert np.allclose(sdpa.transpose(0, 1).numpy(), expanded, atol=1e-12)


def test_oracle_write_known_answers():
    x = np.array([[3.0, 4.0]])
    assert np.allclose(ora.rms(x, np.array([2.0, 1.0]), 0.0), [[6 / np.sqrt(12.5), 4 / np.sqrt(12.5)]])
    angle = np.array([[0.5, 0.5]])
    assert np.allclose(ora.rope(np.array([[1.0, 0.0]]), np.cos(angle), np.sin(angle)), [[np.cos(0.5), np.sin(0.5)]])
    cache = np.arange(2 * 2 * 1, dtype=float).reshape(2, 2, 1)
    rows, valid = ora.gather(cache, np.array([1, -1]), 3)
    assert rows[:, 0].tolist() == [2, 3, 0] and valid.tolist() == [True, True, False]
