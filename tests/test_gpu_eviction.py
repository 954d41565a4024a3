"""Accumulated attention weights against float64, and eviction against a plain
program, bit for bit: every weight, kept position and byte of the cache.

Bounds of the weights: a weight is exp of a score less a log sum.  A dot of D products
is off by at most (D + 4) 2^-24 sum |q_i k_i|, the scaled score and the log sum in
powers of two by a few 2^-24 of each, the exponential and each addition by 2^-24 of
theirs (``oracle.eviction.added_weights`` adds these up, doubled)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import eviction, paged
from oracle import eviction as oracle
from oracle import paged as paged_oracle
from test_gpu_paged import BF16, F16, FP8, Case, _f64
from test_gpu_paged_fp4 import FP4, Case4

pytestmark = pytest.mark.gpu


def _case(device, seed, lengths, chunks, heads, kv_heads, dim, page, dtype, **kw):
    if dtype == FP4:
        return Case4(device, seed, lengths, chunks, heads, kv_heads, dim, page, **kw)
    return Case(device, seed, lengths, chunks, heads, kv_heads, dim, page, dtype, **kw)


WEIGHTS = [
    # lengths, chunks, heads, kv_heads, dim, page, dtype
    ([1], [1], 1, 1, 64, 1, BF16),
    ([1, 2, 31, 32, 65], [1] * 5, 4, 2, 128, 16, BF16),
    ([129, 0, 700], [1, 1, 1], 8, 2, 128, 64, F16),
    ([300, 77], [1, 1], 8, 8, 64, 32, FP8),
    ([513, 64], [1, 1], 6, 1, 256, 16, BF16),
    ([95, 130], [1, 1], 40, 1, 128, 4, FP4),
    ([40, 70, 9], [5, 0, 9], 7, 1, 64, 16, F16),     # an odd group, an empty chunk, a whole sequence
    ([3, 50], [6, 2], 4, 4, 128, 16, BF16),          # more new tokens than keys: early rows see nothing
    ([0, 0], [2, 3], 4, 2, 64, 16, FP8),             # nothing cached at all
    ([260], [130], 6, 2, 128, 16, FP4),              # rows in several stages
    ([200, 517, 90], [200, 33, 1], 8, 2, 128, 32, FP8),
    ([170, 301], [64, 129], 5, 1, 256, 64, FP4),
    ([700], [700], 16, 1, 128, 16, BF16),            # rows in pieces
    ([900, 300], [900, 20], 12, 2, 64, 16, FP4),
    ([333], [300], 8, 2, 256, 16, FP8),
    ([2000], [64], 4, 4, 128, 64, F16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,dtype", WEIGHTS)
def test_weights(device, lengths, chunks, heads, kv_heads, dim, page, dtype, causal) -> None:
    print(f"weights {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} {dtype} {causal}", flush=True)
    c = _case(device, 5 + dim, lengths, chunks, heads, kv_heads, dim, page, dtype)
    q, args = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, *args, causal=causal, return_lse=True)
    weights = eviction.new_weights(c.cache)
    weights += torch.rand(weights.shape, generator=torch.Generator().manual_seed(1)).to(device)
    before = weights.double().cpu().numpy()
    eviction.accumulate_weights(weights, q, c.cache, *args[:2], lse, args[2], causal=causal)
    want, off = oracle.added_weights(_f64(c.q), np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts,
                                     lse.double().cpu().numpy(), dim**-0.5, causal=causal)
    got = weights.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert np.array_equal(got[off == 0], before[off == 0])  # rows of no sequence
    assert (np.abs(got - before - want) <= off + 2.0**-23 * (np.abs(before) + want)).all()
    again = eviction.new_weights(c.cache)
    eviction.accumulate_weights(again, q, c.cache, *args[:2], lse, args[2], causal=causal)
    once = again.clone()
    again.zero_()
    eviction.accumulate_weights(again, q, c.cache, *args[:2], lse, args[2], causal=causal)
    assert torch.equal(again, once)
    if causal and min(lengths) > 0 and all(a >= b for a, b in zip(lengths, chunks)):  # every row's weights add up to 1
        total = sum(chunks) * heads // kv_heads
        assert (once.double().sum(1) - total).abs().max() <= 2.0**-10 * total


def test_weights_of_uniform_chunks_and_padded_batches(device) -> None:
    """Without starts as with them; tokens of no sequence add nothing."""

    c = _case(device, 9, [90, 200, 64], [20, 20, 20], 8, 2, 128, 16, BF16)
    q, (table, lengths, starts) = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, table, lengths, return_lse=True)
    weights = [eviction.new_weights(c.cache) for _ in range(3)]
    eviction.accumulate_weights(weights[0], q, c.cache, table, lengths, lse)
    eviction.accumulate_weights(weights[1], q, c.cache, table, lengths, lse, starts)
    nan = torch.full((7, 8, 128), math.nan, dtype=BF16, device=device)
    eviction.accumulate_weights(weights[2], torch.cat([nan, q, nan]), c.cache, table, lengths,
                                torch.cat([nan[:, :, 0].float(), lse, nan[:, :, 0].float()]), starts + 7)
    assert torch.allclose(weights[0], weights[1], rtol=2.0**-18, atol=0)  # the same sums, cut otherwise
    assert torch.allclose(weights[0], weights[2], rtol=2.0**-18, atol=0)


def test_weights_of_shared_pages_are_all_added(device) -> None:
    c = _case(device, 10, [256, 256], [1, 1], 8, 2, 128, 64, BF16)
    table, lengths, _ = c.device_args()
    table[1] = table[0]
    q = c.q.to(device)
    _, lse = paged.attention(q, c.cache, table, lengths, return_lse=True)
    both, one = eviction.new_weights(c.cache), eviction.new_weights(c.cache)
    eviction.accumulate_weights(both, q, c.cache, table, lengths, lse)
    for b in range(2):
        eviction.accumulate_weights(one, q[b:b + 1], c.cache, table[b:b + 1], lengths[b:b + 1], lse[b:b + 1])
    assert torch.allclose(both, one, rtol=2.0**-18, atol=0) and (both > 0).sum() == 2 * 256


def test_weights_do_not_see_what_rows_do_not(device) -> None:
    """A NaN key is NaN in its own weight alone; later tokens' rows and unseen keys
    stay out of each other's sums."""

    c = _case(device, 12, [300], [40], 8, 2, 128, 16, BF16)
    q, args = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, *args, return_lse=True)
    want, got = eviction.new_weights(c.cache), eviction.new_weights(c.cache)
    eviction.accumulate_weights(want, q, c.cache, *args[:2], lse, args[2])
    row = int(paged.cache_rows(c.cache, args[0], torch.tensor([280], device=device), torch.zeros(1, device=device).long()))
    c.cache.keys.view(-1, 2, 128)[row, 1] = math.nan
    eviction.accumulate_weights(got, q, c.cache, *args[:2], lse, args[2])
    assert torch.isnan(got[1, row])
    got[1, row] = want[1, row]
    assert torch.equal(got, want)


def _parts(cache) -> list[torch.Tensor]:
    """The cache's bytes, ``[rows, kv_heads, bytes]`` each."""

    out = []
    for x in (cache.keys, cache.values):
        size = cache.head_dim // 2 if cache.dtype == FP4 else cache.head_dim * x.element_size()
        out.append(x.contiguous().view(torch.uint8).reshape(cache.rows, cache.kv_heads, size))
    for x in (cache.key_scales, cache.value_scales):
        if x is not None and cache.dtype == FP4:
            out.append(x.view(torch.uint8).transpose(1, 2).reshape(cache.rows, cache.kv_heads, -1))
        elif x is not None:
            out.append(x.reshape(cache.rows, cache.kv_heads, 1).view(torch.uint8))
    return [x.cpu().numpy().copy() for x in out]


def _check_eviction(device, c, weights, keep, recent, per_head) -> None:
    table, lengths, _ = c.device_args()
    parts, before = _parts(c.cache), weights.cpu().numpy().copy()
    out, kept = eviction.evict(c.cache, table, lengths, weights, keep, recent=recent, per_head=per_head)
    want_out, want_kept = oracle.evict(parts, before, c.table.numpy(), c.page, c.lengths, keep, recent, per_head)
    assert out.dtype == torch.int32 and out.tolist() == want_out.tolist()
    assert kept.dtype == torch.int64
    assert np.array_equal(kept.cpu().numpy(), want_kept if per_head else want_kept[:, 0])
    assert np.array_equal(weights.cpu().numpy(), before, equal_nan=True)
    for got, want in zip(_parts(c.cache), parts):
        assert np.array_equal(got, want)
    assert lengths.tolist() == list(c.lengths)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("lengths,kv_heads,dim,page,dtype,keep,recent,layout", [
    ([1], 1, 64, 1, BF16, 1, 0, "nhd"),
    ([2, 1, 0, 5], 2, 64, 1, BF16, 1, 1, "nhd"),
    ([300, 64, 63, 65], 2, 128, 16, BF16, 64, 10, "hnd"),
    ([300, 64, 63, 65], 3, 64, 16, F16, 64, 0, "wide"),
    ([700, 129], 2, 128, 64, FP8, 128, 128, "nhd"),
    ([1500], 4, 256, 8, FP8, 1000, 33, "hnd"),
    ([5000, 4097, 4096], 2, 64, 32, FP4, 4000, 77, "paged"),
    ([9000], 3, 128, 16, FP4, 700, 5, "rows"),
    ([333, 20], 8, 256, 4, FP4, 332, 0, "wide"),
    ([20000, 100, 16385], 2, 64, 64, BF16, 9000, 50, "nhd"),     # lists of several workgroups
    ([40001], 3, 64, 16, FP4, 8192, 8192, "paged"),
    ([17000, 5], 1, 128, 256, FP8, 16999, 1, "hnd"),
    ([400], 8, 128, 16, BF16, 500, 3, "nhd"),        # nothing to evict
])
def test_evict(device, lengths, kv_heads, dim, page, dtype, keep, recent, layout, per_head) -> None:
    print(f"evict {lengths} {kv_heads}x{dim} page {page} {dtype} keep {keep} recent {recent} {layout} {per_head}", flush=True)
    c = _case(device, 3 + dim, lengths, [0] * len(lengths), kv_heads, kv_heads, dim, page, dtype, layout=layout)
    gen = torch.Generator().manual_seed(keep)
    weights = torch.exp(3 * torch.randn(kv_heads, c.cache.rows, generator=gen))
    _check_eviction(device, c, weights.to(device), keep, recent, per_head)


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("n", [6001, 25003])
@pytest.mark.parametrize("kind", ["ties", "zeros", "nan", "signs", "infinite", "near", "rising", "falling"])
def test_evict_by_any_weights(device, kind, n, per_head) -> None:
    """Ties go to the lowest position, also where nothing has any weight; keys whose
    sums overflow or are NaN have their place too."""

    kv_heads = 3
    c = _case(device, 4, [n, 100], [0, 0], kv_heads, kv_heads, 64, 16, BF16)
    gen = torch.Generator().manual_seed(5)
    shape = (kv_heads, c.cache.rows)
    weights = torch.rand(shape, generator=gen)
    if kind == "ties":
        weights = torch.randint(0, 4, shape, generator=gen).float()
    elif kind == "zeros":
        weights = torch.zeros(shape)
    elif kind == "nan":
        weights[torch.rand(shape, generator=gen) < 0.7] = math.nan
    elif kind == "signs":
        weights = (weights - 0.5) * torch.randint(0, 2, shape, generator=gen)  # zeros of both signs
        weights[torch.rand(shape, generator=gen) < 0.1] *= -0.0
    elif kind == "infinite":
        weights[torch.rand(shape, generator=gen) < 0.4] = math.inf
        weights[torch.rand(shape, generator=gen) < 0.2] = 3e38
    elif kind == "near":
        weights = 1 + torch.randint(0, 3, shape, generator=gen) * 2.0**-23
    elif kind in ("rising", "falling"):
        at = torch.zeros(c.cache.rows)
        rows = paged.cache_rows(c.cache, c.table, torch.arange(n), torch.zeros(n, dtype=torch.int64))
        at[rows] = torch.arange(n).float()
        weights = (at if kind == "rising" else -at).expand(shape).contiguous()
    for keep, recent in ((1000, 17), (1, 0), (n - 1, 2), (4096, 4096), (2 * n // 3, 0)):
        _check_eviction(device, c, weights.to(device), keep, recent, per_head)


def test_evicted_keys_past_32_bits(device) -> None:
    page, kv_heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * kv_heads * dim * 2)
    cache = paged.new_cache(pages, page, kv_heads, dim, device=device)
    table = torch.tensor([[pages - 1, 1, pages - 2, 0]], dtype=torch.int32, device=device)
    n = 250
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, kv_heads, dim, generator=gen).to(BF16).to(device) for _ in range(2))
    rows = paged.cache_rows(cache, table, torch.arange(n, device=device), torch.zeros(n, device=device).long())
    paged.append(cache, k, v, rows, torch.zeros(n, device=device).long(), rope_dim=0)
    weights = eviction.new_weights(cache)
    weights[:, rows] = torch.rand(kv_heads, n, generator=gen).to(device)
    want = weights[:, rows].double().sum(0).float().cpu().numpy()
    lengths, kept = eviction.evict(cache, table, torch.tensor([n], dtype=torch.int32, device=device), weights, 100, recent=3)
    assert lengths.tolist() == [100] and kept[0].tolist() == oracle.choose(want, n, 100, 3)
    for got, x in zip(paged.read(cache, rows[:100]), (k, v)):
        assert torch.equal(got, x[kept[0]])


@pytest.mark.parametrize("dtype,per_head", [(BF16, False), (FP4, True), (FP4, False), (FP8, True)])
def test_a_server_with_a_budget(device, dtype, per_head) -> None:
    """Prompts, then decode steps that accumulate weights and evict down to a budget
    now and then: the attention is that over the keys which are left, in every step."""

    batch, heads, kv_heads, dim, page, budget = 2, 8, 2, 64, 16, 96
    cache = paged.new_cache(40, page, kv_heads, dim, dtype=dtype, device=device)
    gen = torch.Generator().manual_seed(7)
    table = torch.randperm(40, generator=gen)[:26].view(2, 13).to(torch.int32).to(device)
    weights = eviction.new_weights(cache)
    alive = [[[] for _ in range(kv_heads)] for _ in range(batch)]  # keys and values in cache order

    def row(n):
        return torch.randn(n, kv_heads, dim, generator=gen).to(cache.row_dtype)

    def add(lengths, counts, first_position):
        total = sum(counts)
        k, v, q = row(total), row(total), torch.randn(total, heads, dim, generator=gen).to(cache.row_dtype)
        at = torch.cat([torch.arange(n, n + m) for n, m in zip(lengths, counts)]).to(device)
        sequence = torch.repeat_interleave(torch.arange(batch), torch.tensor(counts)).to(device)
        rows = paged.cache_rows(cache, table, at, sequence)
        positions = torch.cat([torch.arange(p, p + m) for p, m in zip(first_position, counts)]).to(device)
        q = paged.append(cache, k.to(device), v.to(device), rows, positions, queries=q.to(device))
        stored = [_f64(x) for x in paged.read(cache, rows)]
        for t in range(total):
            for g in range(kv_heads):
                alive[int(sequence[t])][g].append((stored[0][t, g], stored[1][t, g]))
        return q

    def attend(q, lengths, starts):
        dev = torch.tensor(lengths, dtype=torch.int32, device=device)
        first = torch.tensor(starts, dtype=torch.int32, device=device)
        out, lse = paged.attention(q, cache, table, dev, first, return_lse=True)
        eviction.accumulate_weights(weights, q, cache, table, dev, lse, first)
        for b in range(batch):
            for t in range(starts[b], starts[b + 1]):
                for h in range(heads):
                    mine = alive[b][h * kv_heads // heads][:lengths[b] - (starts[b + 1] - 1 - t)]
                    ref, ref_lse, w, _ = paged_oracle.attend(_f64(q)[t, h], np.array([x[0] for x in mine]),
                                                             np.array([x[1] for x in mine]), dim**-0.5)
                    # bf16 output and weights, and an fp8 row read back as bf16 (2^-8 of each element)
                    slack = 2.0**-7 * (np.abs(ref) + w) + (2.0**-4 * w if dtype == FP8 else 0)
                    assert (np.abs(_f64(out)[t, h] - ref) <= slack + 1e-6).all()

    lengths, position = [150, 70], [150, 70]
    q = add([0, 0], lengths, [0, 0])
    attend(q, lengths, [0, 150, 220])
    for step in range(12):
        if step % 5 == 0:
            before = weights.cpu().numpy().copy()
            new, kept = eviction.evict(cache, table, torch.tensor(lengths, dtype=torch.int32, device=device), weights, budget,
                                       recent=8, per_head=per_head)
            kept = kept if per_head else kept[:, None].expand(-1, kv_heads, -1)
            for b in range(batch):
                for g in range(kv_heads):
                    alive[b][g] = [alive[b][g][j] for j in kept[b, g].tolist() if j >= 0]
            assert new.tolist() == [min(n, budget) for n in lengths]
            assert weights.sum() <= before.sum() * (1 + 1e-5)
            lengths = new.tolist()
        counts = [1, 1] if step % 3 else [3, 2]
        q = add(lengths, counts, position)
        lengths, position = ([a + b for a, b in zip(x, counts)] for x in (lengths, position))
        attend(q, lengths, [0, counts[0], sum(counts)])


def test_captured_weights_and_eviction(device) -> None:
    """Both in one graph on a stream of its own, replayed between eager calls."""

    c = _case(device, 14, [900, 300], [200, 10], 8, 2, 128, 16, BF16)
    q, (table, lengths, starts) = c.q.to(device), c.device_args()
    _, lse = paged.attention(q, c.cache, table, lengths, starts, return_lse=True)
    keys, values = c.cache.keys.clone(), c.cache.values.clone()
    weights = eviction.new_weights(c.cache)

    def step():
        c.cache.keys.copy_(keys)
        c.cache.values.copy_(values)
        weights.zero_()
        eviction.accumulate_weights(weights, q, c.cache, table, lengths, lse, starts)
        return eviction.evict(c.cache, table, lengths, weights, 256, recent=20, per_head=True)

    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    with torch.cuda.stream(stream):
        for turn in range(4):
            lse += 0.01 * turn
            want = [x.clone() for x in step()]
            state = [x.clone() for x in (weights, c.cache.keys, c.cache.values)]
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for a, b in zip((weights, c.cache.keys, c.cache.values), state):
                assert torch.equal(a.view(torch.int16) if a.dtype == BF16 else a, b.view(torch.int16) if b.dtype == BF16 else b)


def test_refusals(device) -> None:
    cache = paged.new_cache(4, 16, 2, 128, device=device)
    table = torch.zeros(2, 2, dtype=torch.int32, device=device)
    lengths = torch.ones(2, dtype=torch.int32, device=device)
    q = torch.zeros(2, 4, 128, dtype=BF16, device=device)
    lse = torch.zeros(2, 4, device=device)
    w = eviction.new_weights(cache)
    assert w.shape == (2, 64) and (w == 0).all()

    def refuses(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    add = eviction.accumulate_weights
    refuses("weights must be", add, w[:, :32], q, cache, table, lengths, lse)
    refuses("weights must be", add, w.double(), q, cache, table, lengths, lse)
    refuses("weights must be", add, w.T.contiguous().T, q, cache, table, lengths, lse)
    refuses("one GPU", add, w.cpu(), q, cache, table, lengths, lse)
    refuses("lse", add, w, q, cache, table, lengths, lse[:1])
    refuses("lse", add, w, q, cache, table, lengths, lse.half())
    refuses("lse", add, w, q, cache, table, lengths, lse.cpu())
    refuses("dtype", add, w, q.half(), cache, table, lengths, lse)
    refuses("page_table", add, w, q, cache, table[0], lengths, lse)
    refuses("same number", add, w, q[:1], cache, table, lengths, lse[:1])
    assert add(w, q[:0], cache, table, lengths, lse[:0]) is None
    evict = eviction.evict
    refuses("weights must be", evict, cache, table, lengths, w[:1], 4)
    refuses("page_table", evict, cache, table[0], lengths, w, 4)
    refuses("lengths", evict, cache, table, lengths[:1], w, 4)
    for keep in (0, -1, 1 << 31, 2.5, True, torch.tensor(4)):
        refuses("keep", evict, cache, table, lengths, w, keep)
    for recent in (-1, 5, 1.0):
        refuses("recent", evict, cache, table, lengths, w, 4, recent=recent)
