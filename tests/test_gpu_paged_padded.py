"""Paged attention of batches padded to a fixed number of tokens: the last tokens, or
the first ones, belong to no sequence.  The sequences' own rows are those of the batch
without padding, in every kernel; the others are 0 and their log sums -inf."""

from __future__ import annotations

import functools
import math

import numpy as np
import pytest
import torch

from dsa_amd import paged
from test_gpu_paged import BF16, F16, FP8, Case

pytestmark = pytest.mark.gpu

PADDED = [
    # lengths, chunks, before, after, heads, kv_heads, dim, dtype
    ([300, 40], [1, 1], 0, 6, 8, 2, 128, BF16),                  # a decode step of few sequences in many places
    ([300, 40, 90, 9], [1, 1, 1, 1], 0, 0, 8, 2, 128, BF16),
    ([900, 64, 1, 300], [1, 1, 0, 1], 0, 1, 8, 2, 64, FP8),
    ([700, 515], [50, 50], 0, 100, 8, 2, 128, BF16),             # pieces that another launch joins
    ([700, 515], [50, 50], 7, 93, 8, 2, 128, F16),
    ([900, 64, 1, 300], [70, 1, 1, 30], 0, 154, 8, 2, 64, BF16),
    ([515, 300, 1], [66, 67, 0], 3, 500, 8, 2, 128, FP8),
    ([1000], [30], 0, 34, 8, 2, 256, BF16),                      # one sequence
    ([700], [65], 5, 60, 8, 2, 128, BF16),
    ([1900], [33], 0, 31, 8, 2, 128, F16),
    ([650], [600], 0, 20, 128, 64, 128, BF16),                   # more row tiles than run at a time
    ([650], [300], 0, 320, 128, 64, 128, BF16),
    ([300], [1], 0, 63, 8, 1, 128, BF16),                        # one sequence, most of the batch padding
    ([300], [2], 3, 15, 8, 2, 64, F16),
    ([1300], [1], 0, 40, 8, 2, 128, FP8),
    ([700], [3], 10, 10, 4, 1, 256, BF16),
    ([300], [1], 0, 599, 128, 64, 128, BF16),
    ([300], [0], 0, 64, 8, 1, 128, BF16),                        # nothing but padding
    ([300, 5], [0, 0], 0, 64, 8, 1, 128, BF16),
]


def _padded(c: Case, before: int, after: int, device):
    """Queries and starts of a case with tokens of no sequence around its own."""

    q = torch.full((before + len(c.q) + after, *c.q.shape[1:]), 3.0, dtype=c.q.dtype)
    q[before:before + len(c.q)] = c.q
    return q.to(device), torch.tensor(c.starts + before, dtype=torch.int32, device=device)


@functools.lru_cache(maxsize=1)
def _other_call(device):
    c = Case(device, 93, [3000], [64], 32, 2, 128, 16, BF16)
    return c.q.to(device), c.cache, *c.device_args()


def _soil_memory(device, like) -> None:
    """Leaves numbers of another call's pieces all over the workspace, and NaN where
    the allocator will place the results."""

    paged.attention(*_other_call(device))
    held = [torch.full_like(like, math.nan), torch.full(like.shape[:2], math.nan, device=device)]
    del held


def _check_padding(out, lse, own) -> None:
    for outside in (slice(0, own.start), slice(own.stop, None)):
        assert (out[outside] == 0).all() and (lse[outside] == -math.inf).all()


@pytest.mark.parametrize("lengths,chunks,before,after,heads,kv_heads,dim,dtype", PADDED)
def test_attention_of_padded_batches(device, lengths, chunks, before, after, heads, kv_heads, dim, dtype) -> None:
    print(f"padded: {lengths} {before}+{chunks}+{after} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 91, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    q, starts = _padded(c, before, after, device)
    own = slice(before, before + len(c.q))
    for causal in (True, False):
        _soil_memory(device, q)
        out, lse = paged.attention(q, c.cache, *c.device_args()[:2], starts, causal=causal, return_lse=True)
        c.check(out[own], lse[own], dim**-0.5, causal=causal)
        _check_padding(out, lse, own)


@pytest.mark.parametrize("lengths,chunks,before,after,heads,kv_heads,dim,dtype,k", [
    ([300, 40], [1, 1], 0, 6, 8, 2, 128, BF16, 30),
    ([3000, 700], [2, 1], 2, 5, 8, 2, 128, FP8, 1500),           # lists in pieces
    ([150, 90], [700, 310], 10, 200, 4, 3, 64, BF16, 45),        # a list to a wave
])
def test_selected_attention_of_padded_batches(device, lengths, chunks, before, after, heads, kv_heads, dim, dtype, k) -> None:
    """A list of a token that no sequence has names nothing."""

    print(f"padded lists: {lengths} {before}+{chunks}+{after} {heads}/{kv_heads}x{dim} {dtype} {k}", flush=True)
    heads = heads if heads % kv_heads == 0 else kv_heads
    c = Case(device, 92, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    q, starts = _padded(c, before, after, device)
    own = slice(before, before + len(c.q))
    lists = np.random.default_rng(k).integers(-20, max(lengths) + 20, (len(q), k))
    for b, n in enumerate(lengths):  # no position twice
        for t in range(c.starts[b], c.starts[b + 1]):
            row = lists[before + t]
            row[np.setdiff1d(np.arange(k), np.unique(row, return_index=True)[1])] = -1
    _soil_memory(device, q)
    out, lse = paged.selected_attention(q, c.cache, *c.device_args()[:2], torch.from_numpy(lists).to(device), starts,
                                        return_lse=True)
    c.check(out[own], lse[own], dim**-0.5, lists=lists[own])
    _check_padding(out, lse, own)


@pytest.mark.parametrize("lengths,chunk,heads,kv_heads,dim,dtype", [
    ([900, 300] * 20, 1, 8, 2, 128, BF16),      # a decode step
    ([900, 300] * 40, 1, 8, 2, 64, F16),        # of more sequences than lanes
    ([700, 515], 40, 8, 2, 128, FP8),
    ([300], 20, 8, 2, 256, BF16),
])
def test_starts_that_fall_leave_no_trace(device, lengths, chunk, heads, kv_heads, dim, dtype) -> None:
    """Starts that name tokens again and again have unspecified results, but the next
    call's are what they were."""

    print(f"falling starts: {len(lengths)} x {chunk} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 94, lengths, [chunk] * len(lengths), heads, kv_heads, dim, 16, dtype)
    q = c.q.to(device)
    table, keys, starts = c.device_args()
    want = paged.attention(q, c.cache, table, keys, starts)
    falling = torch.zeros_like(starts)
    falling[1::2] = len(q)                      # 0, T, 0, T, ...
    for bad in (falling, starts.flip(0), starts - 1000, starts + 1000, starts * 1000):
        paged.attention(q, c.cache, table, keys, bad)
        paged.selected_attention(q, c.cache, table, keys, torch.zeros(len(q), 3, dtype=torch.int64, device=device), bad)
        assert torch.equal(paged.attention(q, c.cache, table, keys, starts), want)
