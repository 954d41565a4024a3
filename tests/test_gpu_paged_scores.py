"""Paged attention where the scores lie far from zero, in every kernel: rows whose
best score is hundreds of powers of two below 1, and rows whose first keys score
-inf.  The bounds are those of ``test_gpu_paged``."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import paged
from test_gpu_paged import BF16, F16, FP8, Case

pytestmark = pytest.mark.gpu


def _set_key_dim(c: Case, dim: int, value: float, rows=slice(None)) -> None:
    """Element ``dim`` of every head's key in cache rows ``rows``."""

    raw = c.cache.keys.view(torch.uint8) if c.dtype == FP8 else c.cache.keys
    code = torch.tensor(value, dtype=torch.float32).to(c.dtype)
    flat = raw.view(-1, *raw.shape[2:])
    flat[rows, :, dim] = (code.view(torch.uint8) if c.dtype == FP8 else code).to(raw.device)
    wide = c.keys64.reshape(-1, *c.keys64.shape[2:])
    at = rows if isinstance(rows, slice) else rows.cpu().numpy()
    scale = 1.0 if c.scales[0] is None else c.scales[0].double().numpy().reshape(wide.shape[:2])[at]
    wide[at, :, dim] = code.double().item() * scale
    c.keys64 = wide.reshape(c.keys64.shape)


ROWS = [
    # lengths, chunks, heads, kv_heads, dim, dtype
    ([300, 40], [1, 1], 8, 2, 128, BF16),            # one token
    ([200], [16], 8, 2, 128, BF16),                  # some rows
    ([700], [16], 8, 2, 64, F16),                    # in pieces
    ([333], [20], 8, 2, 128, FP8),
    ([180], [70], 8, 2, 128, BF16),                  # many
    ([900, 300], [200, 77], 8, 2, 64, F16),
    ([400], [150], 4, 2, 128, FP8),
    ([257], [33], 5, 1, 256, BF16),
    ([1000], [30], 8, 2, 256, FP8),
]


@pytest.mark.parametrize("below", [16.0, 80.0, 100.0, 250.0, 4000.0])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,dtype", ROWS)
def test_scores_far_below_zero(device, lengths, chunks, heads, kv_heads, dim, dtype, below) -> None:
    print(f"scores about -{below}: {lengths} {chunks} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 81, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    scale = dim**-0.5
    key = 16.0 if dtype != FP8 else 256.0
    _set_key_dim(c, 0, -key)
    c.q[:, :, 0] = below / scale / (16.0 if dtype != FP8 else 256.0 * 2.0**-6)
    for causal in (True, False):
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
        c.check(out, lse, scale, causal=causal)


@pytest.mark.parametrize("below", [4.0, 60.0, 300.0])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,dtype", [r for r in ROWS if r[-1] != FP8])
def test_first_keys_that_score_minus_infinity(device, lengths, chunks, heads, kv_heads, dim, dtype, below) -> None:
    """Keys with an infinity that the queries weigh negatively have weights of 0, however
    far below zero the later keys' scores are."""

    print(f"-inf, then about -{below}: {lengths} {chunks} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 82, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    scale = dim**-0.5
    _set_key_dim(c, 0, -16.0)
    c.q[:, :, 0] = below / scale / 16.0
    first = [min((3 * n) // 4, n - n_new) for n, n_new in zip(lengths, chunks)]  # every row sees its own key beyond them
    for b, n in enumerate(first):
        rows = paged.cache_rows(c.cache, c.table.to(device), torch.arange(n, device=device),
                                torch.full((n,), b, dtype=torch.int64, device=device))
        flat = c.cache.keys.view(-1, kv_heads, dim)
        flat[rows, :, 0] = -math.inf
    for causal in (True, False):
        lists = np.full((sum(chunks), max(lengths)), -1, dtype=np.int64)
        for b, n in enumerate(lengths):
            for i in range(chunks[b]):
                last = n - chunks[b] + i + 1 if causal else n
                lists[c.starts[b] + i, first[b]:last] = np.arange(first[b], last)
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
        c.check(out, lse, scale, lists=lists)
