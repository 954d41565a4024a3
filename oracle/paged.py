"""Paged key/value cache operators in float64 numpy, one row after the other.

Test infrastructure: the definitions of ``dsa_amd.paged`` (which the reference
has no counterpart of), written without tiling or running sums."""

from __future__ import annotations

import numpy as np

E4M3_MOST = 448.0
LEAST_SCALE = 2.0**-126


def rotate(x: np.ndarray, positions: np.ndarray, rope_dim: int, theta: float) -> np.ndarray:
    """Non-interleaved RoPE of x ``[T, heads, D]``: pairs (i, i + rope_dim / 2)."""

    out = x.astype(np.float64).copy()
    half = rope_dim // 2
    for i in range(half):
        angle = positions.astype(np.float64) * theta ** (-i / half)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        first, second = x[..., i].astype(np.float64), x[..., i + half].astype(np.float64)
        out[..., i] = first * c - second * s
        out[..., i + half] = second * c + first * s
    return out


def head_scale(x: np.ndarray) -> np.ndarray:
    """The scale of each head of an fp8 cache."""

    return np.maximum(np.abs(x).max(axis=-1) / E4M3_MOST, LEAST_SCALE)


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, scale: float):
    """One row over the keys it sees: (output, lse, sum of weights times |value|,
    largest scale * sum |q_i k_i|).  No keys: zeros and -inf."""

    if len(keys) == 0:
        zero = np.zeros(values.shape[-1])
        return zero, -np.inf, zero, 0.0
    scores = (keys @ q) * scale
    top = scores.max()
    weights = np.exp(scores - top)
    total = weights.sum()
    size = scale * (np.abs(keys) @ np.abs(q)).max()
    return weights @ values / total, top + np.log(total), weights @ np.abs(values) / total, size


def attention(q, keys, values, table, lengths, starts, scale, *, causal=True, lists=None):
    """q ``[T, H, D]``; keys and values ``[pages, page_size, G, D]``; ``lists`` the
    positions each token sees (None: its sequence's, up to its own if causal).
    Returns out, lse, weighted |value| and score sizes, for the tests' bounds."""

    tokens, heads, dim = q.shape
    size, kv_heads = keys.shape[1], keys.shape[2]
    out = np.zeros((tokens, heads, dim))
    weighted = np.zeros((tokens, heads, dim))
    lse = np.full((tokens, heads), -np.inf)
    sizes = np.zeros((tokens, heads))
    for b in range(len(lengths)):
        count = starts[b + 1] - starts[b]
        for i in range(count):
            t = starts[b] + i
            if lists is not None:
                seen = np.array([p for p in lists[t] if 0 <= p < lengths[b]], dtype=np.int64)
            else:
                seen = np.arange(max(0, lengths[b] - count + i + 1) if causal else lengths[b])
            page, slot = table[b][seen // size], seen % size
            for h in range(heads):
                g = h * kv_heads // heads
                out[t, h], lse[t, h], weighted[t, h], sizes[t, h] = attend(q[t, h], keys[page, slot, g],
                                                                           values[page, slot, g], scale)
    return out, lse, weighted, sizes
