"""The order of rotated values: projections stored for rotation in adjacent pairs are used with halves after a permutation
(no GPU needed)."""

from __future__ import annotations

import numpy as np

from oracle import latent as ora


def test_adjacent_pairs_permuted_to_halves_keep_the_scores():
    rng = np.random.default_rng(0)
    hidden, d, n = 12, 8, 5
    wq, wk = rng.normal(size=(d, hidden)), rng.normal(size=(d, hidden))
    xq, xk = rng.normal(size=(n, hidden)), rng.normal(size=(n, hidden))
    angle = rng.uniform(0, 6, size=(n, 1)) * 10.0 ** -np.arange(0, d, 2)

    def pairs(x):
        a, b = x[:, ::2], x[:, 1::2]
        return np.stack([a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)], -1).reshape(n, d)

    order = np.r_[0:d:2, 1:d:2]
    both = np.concatenate([angle, angle], 1)

    def halves(x):
        return ora.rope(x, np.cos(both), np.sin(both))

    want = pairs(xq @ wq.T) @ pairs(xk @ wk.T).T
    assert np.allclose(halves(xq @ wq[order].T) @ halves(xk @ wk[order].T).T, want)
