"""Accumulated attention weights of cached keys and eviction by them, in float64
numpy and plain Python.

Test infrastructure: the definitions of ``dsa_amd.eviction`` (which the reference
has no counterpart of)."""

from __future__ import annotations

import numpy as np


def added_weights(q, keys, table, lengths, starts, lse, scale, *, causal=True):
    """q ``[T, H, D]``, keys ``[pages, page_size, G, D]``, lse ``[T, H]``: what each
    cache row's keys ``[G, rows]`` have of the tokens' weights, and a bound on fp32's
    error of it (sums of the products' magnitudes, arguments and additions)."""

    size, kv_heads, dim = keys.shape[1:]
    group = q.shape[1] // kv_heads
    flat = keys.reshape(-1, kv_heads, dim)
    out = np.zeros((kv_heads, len(flat)))
    off = np.zeros((kv_heads, len(flat)))
    eps = 2.0**-24
    for b, n in enumerate(lengths):
        count = starts[b + 1] - starts[b]
        at = np.arange(n)
        rows = table[b][at // size].astype(np.int64) * size + at % size
        last = n - count + np.arange(count) if causal else np.full(count, n - 1)
        seen = at[None] <= np.repeat(last, group)[:, None]
        for g in range(kv_heads):
            mine = slice(g * group, (g + 1) * group)
            x = q[starts[b]:starts[b + 1], mine].reshape(-1, dim)
            sums = lse[starts[b]:starts[b + 1], mine].reshape(-1, 1)
            if not len(x) or not n:
                continue
            k = flat[rows, g]
            p = np.where(seen, np.exp(np.where(seen, scale * (x @ k.T) - np.where(np.isfinite(sums), sums, 0), -np.inf)), 0)
            wide = np.where(seen, abs(scale) * (np.abs(x) @ np.abs(k).T), 0)
            wrong = p * 2 * ((dim + 12) * wide + 3 * np.where(np.isfinite(sums), np.abs(sums), 0) + 8 + len(x)) * eps
            out[g, rows] += p.sum(0)
            off[g, rows] += wrong.sum(0) + len(x) * 2.0**-125
    return out, off


def choose(weights: np.ndarray, n: int, keep: int, recent: int) -> list[int]:
    """Where each of the first min(n, keep) positions' keys were before: the newest
    min(recent, keep) and the largest weights of the others, ties to the lowest."""

    m = min(n, keep)
    if n == m:
        return list(range(n))
    old = n - min(recent, m)
    value = [(-np.inf, 1) if np.isnan(w) else (float(w), 0) for w in weights[:old]]
    chosen = sorted(range(old), key=lambda j: (-value[j][0], value[j][1], j))[:m - (n - old)]
    kept = set(chosen) | set(range(old, n))
    movers = iter(sorted(j for j in kept if j >= m))
    return [j if j in kept else next(movers) for j in range(m)]


def evict(arrays, weights, table, page_size, lengths, keep, recent, per_head):
    """``arrays``: cache parts ``[rows, G, ...]``, changed in place with ``weights``
    ``[G, rows]``; returns the new lengths and the kept positions ``[B, lists, keep]``."""

    kv_heads = weights.shape[0]
    lists = kv_heads if per_head else 1
    kept = np.full((len(lengths), lists, keep), -1, dtype=np.int64)
    for b, n in enumerate(lengths):
        at = np.arange(n)
        rows = table[b][at // page_size].astype(np.int64) * page_size + at % page_size
        for g in range(lists):
            heads = [g] if per_head else list(range(kv_heads))
            with np.errstate(invalid="ignore", over="ignore"):
                mass = weights[heads][:, rows].astype(np.float64).sum(0).astype(np.float32)
            where = np.array(choose(mass, n, keep, recent), dtype=np.int64)
            kept[b, g, :len(where)] = where
            for h in heads:
                moved = weights[h, rows[where]].copy()
                for x in arrays:
                    x[rows[:len(where)], h] = x[rows[where], h].copy()
                if n > keep:
                    weights[h, rows] = 0
                    weights[h, rows[:len(where)]] = moved
    return np.array([min(n, keep) for n in lengths]), kept
