"""Paged attention over the batches that its variants split between them: few and
many rows a sequence in one batch, more sequences than a wave has lanes, lists of
many tokens, and caches that hold infinities and NaN where a row does not look.
The bounds are those of ``test_gpu_paged``."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import paged
from test_gpu_paged import BF16, F16, FP8, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,dtype,layout", [
    ([700], [70], 8, 2, 64, 16, BF16, "nhd"),                # 280 rows: two row tiles, keys in pieces
    ([700], [65], 8, 2, 128, 16, BF16, "hnd"),
    ([515, 300], [66, 67], 8, 2, 128, 64, F16, "nhd"),
    ([333], [129], 4, 2, 128, 32, FP8, "nhd"),
    ([400], [150], 3, 3, 64, 8, FP8, "wide"),
    ([257], [33], 5, 1, 256, 16, BF16, "nhd"),
    ([1200], [20], 8, 2, 256, 16, F16, "wide"),
    ([1000], [30], 8, 2, 256, 32, FP8, "hnd"),
    ([900, 64, 1, 300], [200, 1, 1, 70], 8, 2, 128, 16, BF16, "nhd"),   # decode steps beside prefills
    ([900, 640, 130, 33], [1, 20, 130, 3], 6, 2, 64, 16, FP8, "nhd"),
    ([0, 130, 40], [140, 130, 150], 4, 2, 128, 16, BF16, "nhd"),        # rows that see nothing
    ([1900], [31], 8, 2, 128, 16, BF16, "nhd"),              # 124 rows: one below the other variant
    ([1900], [33], 8, 2, 128, 16, BF16, "nhd"),
])
def test_rows_of_every_variant(device, lengths, chunks, heads, kv_heads, dim, page, dtype, layout, causal) -> None:
    print(f"paged rows {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} {dtype} {layout} {causal}", flush=True)
    c = Case(device, 21 + dim, lengths, chunks, heads, kv_heads, dim, page, dtype, layout=layout, hot=True)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
    c.check(out, lse, dim**-0.5, causal=causal)


@pytest.mark.parametrize("chunk,dim,dtype", [(1, 64, BF16), (1, 128, FP8), (9, 64, F16), (40, 64, BF16), (5, 256, BF16)])
def test_more_sequences_than_lanes(device, chunk, dim, dtype) -> None:
    """130 sequences of every length from 0 on, evenly and by starts."""

    print(f"130 sequences of {chunk} tokens, {dim}, {dtype}", flush=True)
    lengths = [(37 * b) % 211 for b in range(130)]
    c = Case(device, 31, lengths, [chunk] * 130, 4, 2, dim, 16, dtype)
    for starts in (True, False):
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(starts), return_lse=True)
        c.check(out, lse, dim**-0.5)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("chunks,heads,kv_heads,dim,dtype", [
    ([1, 1, 1, 1, 1], 8, 2, 128, BF16),
    ([5, 0, 0, 0, 0], 10, 2, 128, BF16),       # 25 rows: two row tiles of one sequence
    ([0, 3, 0, 0, 2], 12, 1, 64, F16),
    ([0, 0, 0, 0, 4], 40, 2, 64, FP8),         # 80 rows
    ([2, 0, 3, 0, 0], 11, 1, 256, FP8),        # an odd group: tiles end inside a token
    ([0, 0, 4, 0, 0], 9, 1, 128, F16),
])
def test_no_more_tokens_than_sequences(device, chunks, heads, kv_heads, dim, dtype, causal) -> None:
    print(f"few tokens {chunks} {heads}/{kv_heads}x{dim} {dtype} {causal}", flush=True)
    for lengths in ([3000, 33, 900, 0, 1700], [3, 2, 1, 65, 2]):
        c = Case(device, 33, lengths, chunks, heads, kv_heads, dim, 16, dtype, hot=True)
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
        c.check(out, lse, dim**-0.5, causal=causal)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 4, 128, FP8), (6, 2, 64, BF16), (4, 4, 64, F16), (32, 2, 128, FP8)])
@pytest.mark.parametrize("chunks", [[1, 1, 1, 1], [2, 0, 1, 1], [3, 2, 1, 0], [2, 2, 2, 2]])
def test_heads_beside_each_other(device, chunks, heads, kv_heads, dim, dtype) -> None:
    """Page tables of more than 128 MiB of cache, whatever the lengths."""

    print(f"heads beside {chunks} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 34, [2100, 40, 700, 0], chunks, heads, kv_heads, dim, 64, dtype, hot=True)
    table, lengths, starts = c.device_args()
    wide = torch.full((4, 2200), 1 << 30, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table
    assert 4 * wide.shape[1] * 64 * kv_heads * 256 >= 128 << 20
    for causal in (True, False):
        out, lse = paged.attention(c.q.to(device), c.cache, wide, lengths, starts, causal=causal, return_lse=True)
        c.check(out, lse, dim**-0.5, causal=causal)


def test_values_that_are_not_finite_beside(device) -> None:
    """The eight-wave variant hides later tokens' values as the others do."""

    c = Case(device, 35, [300], [4], 4, 2, 128, 64, FP8)
    table, lengths, starts = c.device_args()
    wide = torch.full((1, 4200), 1 << 30, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table
    q = c.q.to(device)
    row = int(paged.cache_rows(c.cache, table, torch.tensor([298], device=device), torch.tensor([0], device=device)))
    _poke(c.cache.values, row, [3, 77], 0.0)
    clean = paged.attention(q, c.cache, wide, lengths, starts)
    _poke(c.cache.values, row, [3, 77], math.nan)
    got = paged.attention(q, c.cache, wide, lengths, starts)
    assert torch.equal(got[:2], clean[:2])
    want = clean[2:].float()
    want[:, :, [3, 77]] = math.nan
    assert torch.equal(torch.nan_to_num(got[2:].float(), 7e4), torch.nan_to_num(want, 7e4))


def test_more_uneven_sequences_than_lanes(device) -> None:
    lengths = [(53 * b) % 307 for b in range(100)]
    chunks = [(0, 1, 2, 7, 30, 66)[b % 6] for b in range(100)]
    c = Case(device, 32, lengths, chunks, 4, 1, 64, 16, BF16)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
    c.check(out, lse, 64**-0.5)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,dtype", [
    (1025, 4, 3, 64, BF16),     # 3075 lists: four to a workgroup, the last one short
    (700, 20, 1, 64, FP8),      # two row tiles of a token's heads
    (1030, 4, 2, 128, FP8),
    (1026, 2, 2, 128, F16),
    (600, 2, 2, 256, BF16),
])
def test_lists_of_many_tokens(device, tokens, heads, kv_heads, dim, dtype) -> None:
    print(f"selected, {tokens} tokens {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    heads = heads if heads % kv_heads == 0 else kv_heads
    lengths = [150, 0, 90]
    chunks = [tokens - 310, 10, 300]
    c = Case(device, 41, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    rng = np.random.default_rng(tokens)
    k = 45
    lists = np.full((tokens, k), -1, dtype=np.int64)
    for b, n in enumerate(lengths):
        for t in range(c.starts[b], c.starts[b + 1]):
            m = min(n, int(rng.integers(0, k + 1)))
            lists[t, rng.permutation(k)[:m]] = rng.permutation(n)[:m]
    out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2],
                                        torch.from_numpy(lists).to(device), c.device_args()[2], return_lse=True)
    c.check(out, lse, dim**-0.5, lists=lists)


def _poke(x: torch.Tensor, row: int, dims, value: float) -> None:
    """Sets dims of every head of a cache row."""

    page, slot = divmod(row, x.shape[1])
    if x.dtype == FP8:
        x.view(torch.uint8)[page, slot, :, dims] = 0x7F if math.isnan(value) else 0
    else:
        x[page, slot, :, dims] = value


@pytest.mark.parametrize("length,chunk,heads,kv_heads,dim,dtype", [
    (70, 5, 6, 2, 128, BF16),       # few rows
    (300, 16, 1, 1, 64, F16),
    (90, 3, 8, 2, 256, FP8),
    (200, 30, 8, 2, 128, F16),      # some
    (150, 40, 4, 2, 64, FP8),
    (700, 31, 8, 2, 128, BF16),     # in pieces
    (180, 70, 8, 2, 128, BF16),     # many
    (170, 150, 4, 2, 64, F16),
    (220, 40, 8, 2, 256, FP8),
    (130, 130, 3, 1, 256, BF16),
])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(device, length, chunk, heads, kv_heads, dim, dtype) -> None:
    """A causal row's result does not depend on what later tokens' rows hold: not
    a bit of it, whether they hold zeros, infinities or NaN."""

    print(f"not finite: {length} {chunk} {heads}/{kv_heads}x{dim} {dtype}", flush=True)
    c = Case(device, 51, [length], [chunk], heads, kv_heads, dim, 16, dtype)
    args = c.device_args()
    q = c.q.to(device)
    new = torch.arange(length - chunk, length)
    places = [(int(p), [(7 * i) % dim, (11 * i + 3) % dim], (math.inf, -math.inf, math.nan)[i % 3] if dtype != FP8 else math.nan)
              for i, p in enumerate(new[::3]) if p > 0]
    rows = paged.cache_rows(c.cache, args[0], new.to(device), torch.zeros(len(new), dtype=torch.int64, device=device)).tolist()
    row_of = dict(zip(new.tolist(), rows))
    for p, dims, _ in places:
        _poke(c.cache.values, row_of[p], dims, 0.0)
    clean, lse = paged.attention(q, c.cache, *args, return_lse=True)
    for p, dims, value in places:
        _poke(c.cache.values, row_of[p], dims, value)
    got, got_lse = paged.attention(q, c.cache, *args, return_lse=True)
    want = clean.float().clone()
    for p, dims, value in places:
        want[p - (length - chunk):, :, dims] += value
    assert torch.equal(torch.nan_to_num(got.float(), 7e4, 8e4, -8e4), torch.nan_to_num(want, 7e4, 8e4, -8e4))
    assert torch.equal(got_lse, lse)

    # A key, and an fp8 row's scale, that is not finite reaches all of a row.
    for p, dims, _ in places:
        _poke(c.cache.values, row_of[p], dims, 0.0)
    last = int(new[-1])
    if chunk > 1:
        _poke(c.cache.keys, row_of[last], [0], math.nan)
        if dtype == FP8:
            page, slot = divmod(row_of[last], 16)
            c.cache.value_scales[page, slot] = math.inf
            c.cache.key_scales[page, slot] = math.nan
        got = paged.attention(q, c.cache, *args)
        assert torch.equal(got[:-1], clean[:-1])
        assert not torch.isfinite(got[-1]).any()


def test_scales_of_rows_that_no_list_names(device) -> None:
    """Padding entries read position 0, whose scales may hold anything."""

    c = Case(device, 61, [200], [1], 8, 2, 128, 16, FP8)
    lists = np.full((1, 50), -1, dtype=np.int64)
    lists[0, ::2] = np.arange(3, 128, 5)
    page = int(c.table[0, 0])
    c.cache.value_scales[page, 0] = math.inf
    c.cache.key_scales[page, 0] = math.nan
    out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2],
                                        torch.from_numpy(lists).to(device), return_lse=True)
    c.check(out, lse, 128**-0.5, lists=lists)


@pytest.mark.parametrize("length,chunk,heads,kv_heads,dim,dtype,causal", [
    (1300, 1152, 64, 32, 64, BF16, True),      # nine row tiles of 256 rows where eight run at a time
    (1300, 1152, 64, 32, 64, FP8, False),
    (650, 600, 128, 64, 128, F16, True),       # five, four at a time: more room than keys for the last one
    (2000, 800, 128, 64, 128, BF16, True),     # seven: three left over
    (700, 530, 64, 64, 256, BF16, True),       # five of 128 rows
    (600, 512, 64, 64, 256, FP8, True),        # four: none left over
    (20, 600, 128, 64, 64, BF16, True),        # more tokens than keys
    (0, 600, 128, 64, 64, BF16, True),
    (300, 280, 256, 128, 64, F16, True),       # three, two at a time
])
def test_more_row_tiles_than_workgroups(device, length, chunk, heads, kv_heads, dim, dtype, causal) -> None:
    """One sequence whose row tiles do not divide by the workgroups that run at a
    time; the first and the last kv head are checked."""

    print(f"row tiles {length} {chunk} {heads}/{kv_heads}x{dim} {dtype} {causal}", flush=True)
    c = Case(device, 71, [length], [chunk], heads, kv_heads, dim, 16, dtype)
    outs = [paged.attention(c.q.to(device), c.cache, *c.device_args(starts), causal=causal, return_lse=True)
            for starts in (True, False)]
    group = heads // kv_heads
    keep = [*range(group), *range(heads - group, heads)]
    c.q, c.heads = c.q[:, keep], 2 * group
    c.keys64, c.values64 = c.keys64[:, :, [0, -1]], c.values64[:, :, [0, -1]]
    for out, lse in outs:
        c.check(out[:, keep], lse[:, keep], dim**-0.5, causal=causal)
