"""e4m3 rows with a scale for every 128 columns and their product, in float64 (no reference file:
the formulas are those of ``slipstream_amd.kernels.quantize_fp8`` and ``fp8_gemm``)."""

from __future__ import annotations

import numpy as np

BLOCK = 128
TOP = 448.0
SMALLEST = TOP * 2.0**-126


def e4m3(v: np.ndarray) -> np.ndarray:
    """float64 values of magnitude at most 448 -> the nearest e4m3 value, half to even."""
    _, e = np.frexp(v)  # |v| = f 2^e, f in [0.5, 1)
    step = np.exp2(np.maximum(e, -5) - 4.0)  # three bits behind the first one; below 2^-6 those of 2^-6
    return np.rint(v / step) * step


def quantize_rows(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """``[m, k]`` -> (e4m3 values ``[m, k]``, scales ``[m, ceil(k / 128)]`` as fp32 division gives them)."""
    m, k = x.shape
    q = np.zeros((m, k))
    scale = np.zeros((m, -(-k // BLOCK)), dtype=np.float32)
    for b in range(scale.shape[1]):
        part = x[:, b * BLOCK : (b + 1) * BLOCK]
        top = np.abs(part).max(axis=1)
        bad = ~np.isfinite(part).all(axis=1)
        live = (top >= SMALLEST) & ~bad
        safe = np.where(live, top, 1.0)[:, None]
        q[:, b * BLOCK : (b + 1) * BLOCK] = np.where(live[:, None], e4m3(np.where(live[:, None], part, 0) * TOP / safe), 0)
        scale[:, b] = np.where(live, safe[:, 0].astype(np.float32) / np.float32(TOP), 0)
        scale[bad, b] = np.nan
    return q, scale


def widen(scale: np.ndarray, rows: int | None, cols: int) -> np.ndarray:
    """A scale for each value: blocks of 128 columns and, with ``rows``, of 128 rows."""
    s = np.repeat(scale.astype(np.float64), BLOCK, axis=1)[:, :cols]
    return s if rows is None else np.repeat(s, BLOCK, axis=0)[:rows]


def gemm(q: np.ndarray, scale: np.ndarray, w: np.ndarray, w_scale: np.ndarray,
         bias: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
    """The product, and the sum of its terms' magnitudes (what rounding errors go by)."""
    x = q * widen(scale, None, q.shape[1])
    y = w * widen(w_scale, w.shape[0], w.shape[1])
    out = x @ y.T
    size = np.abs(x) @ np.abs(y).T
    return (out, size) if bias is None else (out + bias, size + np.abs(bias))
