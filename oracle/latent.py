"""Attention over latents and the latent cache's write in float64 (no reference file: the formulas are
those of ``slipstream_amd.kernels.latent_attention`` and ``latent_cache``; the causal rule and the edge
rules are those of ``slipstream/kernels/attention_ref.py:42-89`` and ``triton_paged.py:133-206``)."""

from __future__ import annotations

import numpy as np


def rope(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    a, b = np.split(x, 2, axis=-1)
    return x * cos + np.concatenate([-b, a], axis=-1) * sin


def rms(x: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * weight


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, valid: np.ndarray, length: int,
           scale: float) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """``q [n, H, D]`` over ``keys [S, D]`` (or ``[S, H, D]``) and ``values``: query j sees the valid
    keys i <= length - n + j. Returns the output, the sum of p |v| and that of |q| |k|'s largest value
    (what rounding errors go by)."""
    n, heads, _ = q.shape
    s_n = keys.shape[0]
    if keys.ndim == 2:
        keys = np.repeat(keys[:, None], heads, axis=1)
        values = np.repeat(values[:, None], heads, axis=1)
    out = np.zeros((n, heads, values.shape[2]))
    size, reach = np.zeros_like(out), np.zeros((n, heads, 1))
    for j in range(n):
        sees = valid & (np.arange(s_n) <= length - n + j)
        if not sees.any():
            continue
        k, v = keys[sees], values[sees]
        s = np.einsum("hd,shd->hs", q[j], k) * scale
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[j] = np.einsum("hs,shd->hd", p, v)
        size[j] = np.einsum("hs,shd->hd", p, np.abs(v))
        reach[j, :, 0] = np.einsum("hd,shd->hs", np.abs(q[j]), np.abs(k)).max(axis=1) * abs(scale)
    return out, size, reach


def gather(cache: np.ndarray, table: np.ndarray, length: int) -> tuple[np.ndarray, np.ndarray]:
    """``cache [num_blocks, block_size, W]`` -> the rows of the sequence's tokens that the table reaches,
    and whether their page is there."""
    nb, bs, width = cache.shape
    n = min(max(length, 0), len(table) * bs)
    rows, valid = np.zeros((n, width)), np.zeros(n, dtype=bool)
    for i in range(n):
        e = int(table[i // bs])
        if 0 <= e < nb:
            rows[i], valid[i] = cache[e, i % bs], True
    return rows, valid
