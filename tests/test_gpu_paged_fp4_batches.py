"""Batches of the 4-bit cache, of accumulated weights and of eviction as servers make
them: padded to a fixed number of tokens, one long chunk among single tokens, and calls
of several launches captured in graphs that share a workspace.  Bounds as in
``test_gpu_paged`` and ``test_gpu_eviction``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dsa_amd import eviction, paged
from oracle import eviction as oracle
from test_gpu_eviction import _case, _check_eviction
from test_gpu_paged import BF16, F16, FP8, _f64
from test_gpu_paged_fp4 import FP4, Case4
from test_gpu_paged_padded import _check_padding, _padded, _soil_memory

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,chunks,before,after,heads,kv_heads,dim", [
    ([300, 40], [1, 1], 0, 6, 8, 2, 128),
    ([900, 64, 1, 300], [1, 1, 0, 1], 0, 1, 8, 2, 64),
    ([700, 515], [50, 50], 7, 93, 8, 2, 128),
    ([900, 64, 1, 300], [70, 1, 1, 30], 0, 154, 8, 2, 64),
    ([700], [65], 5, 60, 8, 2, 256),
    ([1300], [1], 0, 40, 8, 2, 128),
    ([300], [0], 0, 64, 8, 1, 256),
])
def test_attention_of_padded_batches(device, lengths, chunks, before, after, heads, kv_heads, dim) -> None:
    print(f"padded: {lengths} {before}+{chunks}+{after} {heads}/{kv_heads}x{dim}", flush=True)
    c = Case4(device, 95, lengths, chunks, heads, kv_heads, dim, 16)
    q, starts = _padded(c, before, after, device)
    own = slice(before, before + len(c.q))
    for causal in (True, False):
        _soil_memory(device, q)
        out, lse = paged.attention(q, c.cache, *c.device_args()[:2], starts, causal=causal, return_lse=True)
        c.check(out[own], lse[own], dim**-0.5, causal=causal)
        _check_padding(out, lse, own)


@pytest.mark.parametrize("lengths,chunks,before,after,heads,kv_heads,dim,k", [
    ([300, 40], [1, 1], 0, 6, 8, 2, 128, 30),
    ([3000, 700], [2, 1], 2, 5, 8, 2, 64, 1500),
    ([150, 90], [700, 310], 10, 200, 6, 3, 256, 45),
])
def test_selected_attention_of_padded_batches(device, lengths, chunks, before, after, heads, kv_heads, dim, k) -> None:
    print(f"padded lists: {lengths} {before}+{chunks}+{after} {heads}/{kv_heads}x{dim} {k}", flush=True)
    c = Case4(device, 96, lengths, chunks, heads, kv_heads, dim, 16)
    q, starts = _padded(c, before, after, device)
    own = slice(before, before + len(c.q))
    lists = np.random.default_rng(k).integers(-20, max(lengths) + 20, (len(q), k))
    for row in lists:  # no position twice
        row[np.setdiff1d(np.arange(k), np.unique(row, return_index=True)[1])] = -1
    _soil_memory(device, q)
    out, lse = paged.selected_attention(q, c.cache, *c.device_args()[:2], torch.from_numpy(lists).to(device), starts,
                                        return_lse=True)
    c.check(out[own], lse[own], dim**-0.5, lists=lists[own])
    _check_padding(out, lse, own)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,dim,group", [(BF16, 128, 4), (F16, 64, 3), (FP8, 256, 4), (FP4, 128, 7), (FP4, 64, 4),
                                             (FP4, 256, 1)])
def test_weights_of_a_chunk_among_single_tokens(device, dtype, dim, group, causal) -> None:
    """A sequence of far more rows than the others, and one of thousands of keys."""

    print(f"weights of a chunk among tokens: {dtype} {dim} {group} {causal}", flush=True)
    lengths = [700, 4500] + [33, 1, 300] * 6
    chunks = [150, 1] + [1, 1, 1] * 6
    kv_heads = 2
    c = _case(device, 97, lengths, chunks, group * kv_heads, kv_heads, dim, 16, dtype)
    q, args = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, *args, causal=causal, return_lse=True)
    weights = eviction.new_weights(c.cache)
    eviction.accumulate_weights(weights, q, c.cache, *args[:2], lse, args[2], causal=causal)
    want, off = oracle.added_weights(_f64(c.q), np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts,
                                     lse.double().cpu().numpy(), dim**-0.5, causal=causal)
    assert (np.abs(weights.double().cpu().numpy() - want) <= off).all()
    again = eviction.new_weights(c.cache)
    eviction.accumulate_weights(again, q, c.cache, *args[:2], lse, args[2], causal=causal)
    assert torch.equal(again, weights)


@pytest.mark.parametrize("lengths,chunks,group,kv_heads,dim,dtype", [
    # more sequences than threads, chunks of some, one that has more tokens than keys, one that has no keys
    ([20 + b % 7 for b in range(300)] + [700, 30, 0, 90] + [20] * 300 + [300], [1] * 300 + [80, 60, 70, 90] + [0, 1, 1] * 100 + [17],
     4, 2, 64, BF16),
    ([20 + b % 7 for b in range(300)] + [700, 30, 0, 90] + [20] * 300 + [300], [1] * 300 + [80, 60, 70, 90] + [0, 1, 1] * 100 + [17],
     4, 2, 128, FP4),
    ([1000, 10] * 8, [70, 1] * 8, 1, 64, 64, F16),          # tiles enough without pieces of rows
    ([1000, 10] * 8, [70, 1] * 8, 1, 64, 64, FP8),
    ([100, 90, 80], [64, 1, 2], 1, 2, 128, BF16),           # as many rows as stay in the kernel of few
    ([100, 90, 80], [65, 1, 2], 1, 2, 128, BF16),           # and one more
    ([900, 5000, 300, 1], [900, 1, 200, 1], 8, 2, 128, FP4),  # most rows a chunk's
    ([9, 300, 700], [0, 0, 600], 3, 2, 64, BF16),
])
def test_weights_of_chunks_among_single_tokens(device, lengths, chunks, group, kv_heads, dim, dtype) -> None:
    print(f"weights of chunks among tokens: {len(lengths)} x {group}/{kv_heads}x{dim} {dtype}", flush=True)
    c = _case(device, 100, lengths, chunks, group * kv_heads, kv_heads, dim, 16, dtype)
    q, args = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, *args, return_lse=True)
    weights = eviction.new_weights(c.cache)
    want, off = oracle.added_weights(_f64(c.q), np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts,
                                     lse.double().cpu().numpy(), dim**-0.5)
    first = None
    for _ in range(3):
        weights.zero_()
        eviction.accumulate_weights(weights, q, c.cache, *args[:2], lse, args[2])
        assert (np.abs(weights.double().cpu().numpy() - want) <= off).all()
        first = weights.clone() if first is None else first
        assert torch.equal(weights, first)


@pytest.mark.parametrize("lengths,chunk,group,kv_heads,dim,dtype,starts", [
    ([4160], 1, 4, 2, 128, FP4, False),
    ([700, 0, 5000, 33], 1, 4, 2, 64, BF16, False),
    ([9000] + [3] * 1099, 1, 1, 8, 64, BF16, False),      # more keys than a sequence's workgroups take at once
    ([9000] + [3] * 1099, 1, 1, 8, 128, FP4, True),
    ([900], 300, 4, 2, 128, FP8, False),                  # pieces of rows
    ([900, 90, 3000], 40, 4, 2, 64, FP4, False),
    ([700] + [2] * 599, 2, 33, 8, 64, F16, False),        # more tiles than a sequence's workgroups
    ([900, 90, 3000], 40, 4, 2, 256, BF16, True),
])
def test_weights_with_room_for_more(device, lengths, chunk, group, kv_heads, dim, dtype, starts) -> None:
    """The same bits whatever the page table has room for; page ids past the lengths are
    any."""

    print(f"weights with room: {len(lengths)} x {chunk} x {group}/{kv_heads}x{dim} {dtype} {starts}", flush=True)
    c = _case(device, 102, lengths, [chunk] * len(lengths), group * kv_heads, kv_heads, dim, 16, dtype)
    q, (table, keys, first) = c.q.to(device), c.device_args()
    first = first if starts else None
    _, lse = paged.attention(q, c.cache, table, keys, first, return_lse=True)
    want, off = oracle.added_weights(_f64(c.q), np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts,
                                     lse.double().cpu().numpy(), dim**-0.5)
    weights = eviction.new_weights(c.cache)
    eviction.accumulate_weights(weights, q, c.cache, table, keys, lse, first)
    assert (np.abs(weights.double().cpu().numpy() - want) <= off).all()
    for room in (20000, 1 << 17):
        more = room // 16 - table.shape[1]
        wide = torch.cat([table, torch.randint(-5, 1 << 30, (len(lengths), more), dtype=torch.int32, device=device)], 1)
        again = eviction.new_weights(c.cache)
        eviction.accumulate_weights(again, q, c.cache, wide, keys, lse, first)
        assert torch.equal(again, weights)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("lengths,kv_heads,page,dtype,room,keep,recent", [
    ([300, 64, 63, 65], 2, 16, BF16, 40000, 64, 10),             # short lists, room for long ones
    ([5000, 4097, 4096], 2, 32, FP4, 1 << 20, 4000, 77),
    ([16384, 16385, 0, 40000, 9000], 2, 64, BF16, 1 << 17, 5000, 9),
    ([30000, 16390, 20], 1, 16, FP8, 30016, 30000, 0),           # long, and nothing to evict
    ([3] * 150 + [17000] + [5, 2, 9] * 200 + [16500, 1, 25000], 2, 4, FP4, 30000, 4, 1),  # more lists than threads
])
def test_eviction_with_room_for_more(device, lengths, kv_heads, page, dtype, room, keep, recent, per_head) -> None:
    """Each list by its own length, whatever the page table has room for; page ids past
    the lengths are any."""

    print(f"room for {room}: {len(lengths)} x {kv_heads} {dtype} keep {keep} {per_head}", flush=True)
    c = _case(device, 101, lengths, [0] * len(lengths), kv_heads, kv_heads, 64, page, dtype)
    more = -(-room // page) - c.table.shape[1]
    gen = torch.Generator().manual_seed(7)
    if more > 0:
        c.table = torch.cat([c.table, torch.randint(-5, 1 << 30, (len(lengths), more), generator=gen, dtype=torch.int32)], 1)
    weights = torch.randint(0, 1000, (kv_heads, c.cache.rows), generator=gen) * 0.125
    _check_eviction(device, c, weights.to(device), keep, recent, per_head)


def test_lengths_beyond_a_small_cache(device) -> None:
    """More keys than the cache has rows: unspecified results, and the next call's are
    what they should be."""

    cache = paged.new_cache(20, 16, 2, 64, device=device)
    cache.keys.zero_(), cache.values.zero_()
    table = torch.zeros(2, 2000, dtype=torch.int32, device=device)
    weights = eviction.new_weights(cache)
    for n in (20000, 16384, 1 << 30, -5):
        lengths = torch.tensor([n, 3], dtype=torch.int32, device=device)
        out, _ = eviction.evict(cache, table, lengths, weights, 64, recent=3, per_head=True)
        assert out.tolist() == [max(0, min(n, 64)), 3]
    table[0, :20] = torch.arange(20)
    weights[:] = torch.arange(320, device=device).flip(0)
    out, kept = eviction.evict(cache, table[:1], torch.tensor([320], dtype=torch.int32, device=device), weights, 64)
    assert out.tolist() == [64] and kept[0].tolist() == list(range(64))


@pytest.mark.parametrize("dtype", [BF16, FP4])
def test_captured_calls_that_share_a_workspace(device, dtype) -> None:
    """A step of lists of several workgroups and one of short lists, captured on one
    stream, replayed in turn with eager calls of the other between them."""

    cases = [_case(device, 98, [20000, 17000], [1, 1], 4, 2, 64, 64, dtype),
             _case(device, 99, [900, 300, 40], [200, 10, 1], 4, 2, 64, 16, dtype)]
    keeps = [9000, 256]
    given, steps = [], []
    for c, keep in zip(cases, keeps):
        q, (table, lengths, starts) = c.q.to(device), c.device_args()
        _, lse = paged.attention(q, c.cache, table, lengths, starts, return_lse=True)
        weights = eviction.new_weights(c.cache)
        tensors = [x.view(torch.uint8) if x.element_size() == 1 else x.view(torch.int16)
                   for x in (c.cache.keys, c.cache.values, c.cache.key_scales, c.cache.value_scales) if x is not None]
        first = [x.clone() for x in tensors]
        given.append((lse, weights, tensors))

        def step(c=c, q=q, table=table, lengths=lengths, starts=starts, lse=lse, weights=weights, tensors=tensors,
                 first=first, keep=keep):
            for x, y in zip(tensors, first):
                x.copy_(y)
            weights.zero_()
            eviction.accumulate_weights(weights, q, c.cache, table, lengths, lse, starts)
            return eviction.evict(c.cache, table, lengths, weights, keep, recent=20)

        steps.append(step)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs, got = [], []
    for step in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            got.append(step())
    with torch.cuda.stream(stream):
        for turn in range(4):
            for i in (0, 1) if turn % 2 else (1, 0):
                lse, weights, tensors = given[i]
                lse += 0.01 * turn
                want = [x.clone() for x in steps[i]()]
                state = [x.clone() for x in (weights, *tensors)]
                steps[1 - i]()
                stream.synchronize()
                graphs[i].replay()
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got[i], want))
                assert all(torch.equal(a, b) for a, b in zip((weights, *tensors), state))
