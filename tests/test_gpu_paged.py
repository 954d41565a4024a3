"""The paged key/value cache against float64: append (rotation, fp8 codes and
scales, skipped rows), attention of one token or a chunk over the cache, and
attention over selected positions.

Bounds.  With u the unit roundoff of the rows' type (2^-8 bf16, 2^-11 fp16), an
output element may be off by its own rounding, u |out|, by the rounding of the
weights, u sum_j w_j |v_j|, and by fp32 errors of the scores: a dot of D
products is off by at most (D + 4) 2^-24 sum |q_i k_i|, the power of two and its
argument by a few 2^-24 more, which a weight sees as a relative error (twice:
numerator and denominator).  The log sum sees the scores' error and n 2^-24 of
its sum.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import decode, paged
from oracle import paged as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _f64(x: torch.Tensor) -> np.ndarray:
    return x.detach().float().cpu().double().numpy()


class Case:
    """A cache whose pages are scattered, rows past every length and unused pages
    holding NaN, and page ids past the last used column out of range."""

    def __init__(self, device, seed, lengths, chunks, heads, kv_heads, dim, page, dtype, *, layout="nhd", spare=2,
                 hot=False):
        gen = torch.Generator().manual_seed(seed)
        self.gen, self.device, self.page, self.dtype = gen, device, page, dtype
        self.lengths, self.chunks = lengths, chunks
        self.row = BF16 if dtype == FP8 else dtype
        used = [-(-n // page) for n in lengths]
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=gen)
        columns = max(1, max(used)) + 1
        table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
        table[:, 0] = order[0]  # an empty sequence's first entry is in range as a program would leave it
        first = 0
        written = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(used):
            table[b, :n] = order[first:first + n].to(torch.int32)
            table[b, n:] = 1 << 30
            first += n
            for p in range(lengths[b]):
                written[table[b, p // page].long(), p % page] = True
        if max(used) == 0:
            table[:, 0] = -7
        self.table = table
        shape = (pages, page, kv_heads, dim)
        keys, values = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)
        if hot:
            keys *= 1 + 7 * (torch.rand(shape[:3], generator=gen) < 0.05)[..., None]
        self.scales = [None, None]
        if dtype == FP8:
            self.scales = [(0.5 + torch.rand(shape[:3], generator=gen)) * 2.0**-6 for _ in range(2)]
            keys, values = (64 * x for x in (keys, values))
        keys, values = keys.clamp(-448, 448).to(dtype), values.clamp(-448, 448).to(dtype)
        self.keys64, self.values64 = _f64(keys), _f64(values)
        if dtype == FP8:
            self.keys64 = self.keys64 * self.scales[0].double().numpy()[..., None]
            self.values64 = self.values64 * self.scales[1].double().numpy()[..., None]
        stale = ~written
        keys, values = keys.float(), values.float()
        keys[stale] = math.nan
        values[stale] = math.nan
        keys, values = keys.to(dtype), values.to(dtype)

        def lay(x):
            raw = x.view(torch.uint8) if dtype == FP8 else x
            if layout == "hnd":  # heads outside slots
                raw = raw.permute(0, 2, 1, 3).contiguous().to(device).permute(0, 2, 1, 3)
            elif layout == "wide":  # keys and values side by side, with room between the heads
                store = torch.zeros(*shape[:3], 2 * dim, dtype=raw.dtype, device=device)
                store[..., dim:] = raw.to(device)
                raw = store[..., dim:]
            else:
                raw = raw.to(device)
            return raw.view(FP8) if dtype == FP8 else raw

        self.cache = paged.PagedCache(lay(keys), lay(values), *(None if s is None else s.to(device) for s in self.scales))
        self.starts = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int64)
        self.heads, self.dim = heads, dim
        self.q = torch.randn(int(self.starts[-1]), heads, dim, generator=gen).to(self.row)

    def device_args(self, starts=True):
        t = (self.table.to(self.device), torch.tensor(self.lengths, dtype=torch.int32, device=self.device))
        return (*t, torch.tensor(self.starts, dtype=torch.int32, device=self.device) if starts else None)

    def check(self, got, lse, scale, *, causal=True, lists=None):
        ref, ref_lse, weighted, sizes = oracle.attention(_f64(self.q), self.keys64, self.values64, self.table.numpy(),
                                                         self.lengths, self.starts, scale, causal=causal, lists=lists)
        u, eps = UNIT[self.row], 2.0**-24
        most = max([1, *self.lengths]) if lists is None else max(1, lists.shape[1])
        score = 2 * ((self.dim + 12) * sizes + 8) * eps
        bound = u * np.abs(ref) + (u * (1 + u) + score[..., None]) * weighted + most * 2.0**-30 + 2.0**-133
        out = _f64(got)
        assert np.isfinite(out).all()
        assert (np.abs(out - ref) <= bound).all(), np.max(np.abs(out - ref) - bound)
        empty = np.isinf(ref_lse)
        assert (out[empty] == 0).all()
        if lse is not None:
            l = lse.cpu().double().numpy()
            assert (l[empty] == -np.inf).all()
            off = np.abs(l - np.where(empty, 0, ref_lse))[~empty]
            assert (off <= (score + (most + 16) * eps + 8 * eps * np.abs(np.where(empty, 0, ref_lse)))[~empty]).all()


ATTENTION = [
    # lengths, chunks, heads, kv_heads, dim, page, dtype, layout
    ([1], [1], 1, 1, 64, 1, BF16, "nhd"),
    ([1, 2, 31, 32, 33], [1] * 5, 4, 2, 128, 16, BF16, "nhd"),
    ([129, 0, 700], [1, 1, 1], 8, 2, 128, 64, F16, "hnd"),
    ([300, 77], [1, 1], 8, 8, 64, 32, FP8, "nhd"),
    ([513, 64], [1, 1], 6, 1, 256, 16, BF16, "wide"),
    ([211, 33], [1, 1], 16, 2, 256, 8, FP8, "hnd"),
    ([95, 130], [1, 1], 40, 1, 128, 4, FP8, "wide"),      # 40 heads of one kv head: three row tiles
    ([40, 70, 9], [5, 0, 9], 7, 1, 64, 16, F16, "nhd"),   # an odd group, an empty chunk, a whole sequence
    ([3, 50], [6, 2], 4, 4, 128, 16, BF16, "nhd"),        # more new tokens than keys: early rows see nothing
    ([0, 0], [2, 3], 4, 2, 64, 16, BF16, "nhd"),          # nothing cached at all
    ([260], [130], 6, 2, 128, 16, BF16, "nhd"),           # a chunk of several row tiles
    ([200, 517, 90], [200, 33, 1], 8, 2, 128, 32, F16, "hnd"),
    ([150], [150], 4, 2, 64, 1, FP8, "nhd"),
    ([170, 301], [64, 129], 5, 1, 256, 64, BF16, "nhd"),
    ([140], [70], 12, 2, 256, 16, FP8, "nhd"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,dtype,layout", ATTENTION)
def test_attention(device, lengths, chunks, heads, kv_heads, dim, page, dtype, layout, causal) -> None:
    print(f"paged attention {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} {dtype} {layout} {causal}", flush=True)
    c = Case(device, 5 + dim, lengths, chunks, heads, kv_heads, dim, page, dtype, layout=layout, hot=True)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
    c.check(out, lse, dim**-0.5, causal=causal)


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 16), (FP8, 128, 32), (F16, 64, 64), (FP8, 64, 16)])
def test_decode_longer_than_one_lookup(device, dtype, dim, page) -> None:
    """Pieces of more than 2048 keys, each row's maximum far down its keys."""

    print(f"paged decode, many heads {dtype} {dim} {page}", flush=True)
    lengths = [5003, 2049, 4096]
    c = Case(device, 3, lengths, [1, 1, 1], 400, 400, dim, page, dtype)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(starts=False), scale=0.3, return_lse=True)
    keep = slice(0, 400, 57)
    c.q, c.heads = c.q[:, keep], len(range(0, 400, 57))
    c.keys64, c.values64 = c.keys64[:, :, keep], c.values64[:, :, keep]
    c.check(out[:, keep], lse[:, keep], 0.3)


def test_uniform_chunks_equal_starts(device) -> None:
    c = Case(device, 9, [90, 200, 64], [20, 20, 20], 8, 2, 128, 16, BF16)
    q = c.q.to(device)
    assert torch.equal(paged.attention(q, c.cache, *c.device_args()), paged.attention(q, c.cache, *c.device_args(False)))


def test_rising_scores_and_far_scores(device) -> None:
    """Scores that rise key by key raise the running maximum again and again; one
    key far above or below the others leaves weights of 1 and 0."""

    n, dim = 700, 64
    c = Case(device, 1, [n], [1], 2, 1, dim, 16, BF16)
    ramp = torch.linspace(-60, 60, n).double()
    for order in (torch.arange(n), torch.arange(n).flip(0)):
        keys = torch.zeros(n, dim)
        keys[:, 0] = ramp[order].float()
        flat = c.cache.keys.view(-1, 1, dim)
        rows = paged.cache_rows(c.cache, c.table.to(device), torch.arange(n, device=device),
                                torch.zeros(n, dtype=torch.int64, device=device))
        flat[rows, 0] = keys.to(BF16).to(device)
        for r, k in zip(rows.tolist(), _f64(keys.to(BF16))):
            c.keys64[r // 16, r % 16, 0] = k
        c.q[:] = 0
        c.q[0, 0, 0], c.q[0, 1, 0] = 9.0, -0.25
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), scale=1.0, return_lse=True)
        c.check(out, lse, 1.0)


@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,dtype,k", [
    ([1], [1], 1, 1, 64, 1, BF16, 1),
    ([300, 40], [1, 1], 8, 2, 128, 16, BF16, 64),
    ([300, 4000, 0], [1, 1, 1], 8, 2, 128, 64, F16, 257),
    ([500, 90], [1, 1], 32, 1, 64, 32, FP8, 100),     # two row tiles of one token's heads
    ([90, 33, 7], [40, 0, 7], 6, 2, 256, 16, BF16, 30),
    ([400], [9], 12, 4, 256, 8, FP8, 333),
    ([5000], [1], 4, 4, 128, 16, FP8, 4500),           # pieces past one lookup's reach at few splits
])
def test_selected(device, lengths, chunks, heads, kv_heads, dim, page, dtype, k) -> None:
    print(f"selected attention {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} {dtype} k {k}", flush=True)
    c = Case(device, 11 + k, lengths, chunks, heads, kv_heads, dim, page, dtype, hot=True)
    tokens = sum(chunks)
    lists = np.full((tokens, k), -1, dtype=np.int64)
    rng = np.random.default_rng(k)
    for b, n in enumerate(lengths):
        for t in range(c.starts[b], c.starts[b + 1]):
            m = min(n, int(rng.integers(0, k + 1)) if t % 3 else k)
            chosen = rng.permutation(n)[:m]
            at = rng.permutation(k)[:m]       # padding anywhere in the list
            lists[t, at] = chosen
            junk = np.flatnonzero(lists[t] < 0)[::2]
            lists[t, junk] = rng.choice([-1, -5, n, n + 1000000, 2**40, -2**62], len(junk))
    if tokens > 1:
        lists[-1] = -1                        # a list of padding alone
    wide = torch.full((tokens, k + 3), -9, dtype=torch.int64)
    wide[:, :k] = torch.from_numpy(lists)
    out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2], wide.to(device)[:, :k],
                                        c.device_args()[2], return_lse=True)
    c.check(out, lse, dim**-0.5, lists=lists)


def test_selected_keys_that_hold_nan_elsewhere(device) -> None:
    """Rows that no list names may hold anything, position 0 among them."""

    c = Case(device, 2, [200], [1], 8, 2, 128, 16, BF16)
    flat_k, flat_v = c.cache.keys.view(-1, 2, 128), c.cache.values.view(-1, 2, 128)
    rows = paged.cache_rows(c.cache, c.table.to(device), torch.arange(200, device=device),
                            torch.zeros(200, dtype=torch.int64, device=device))
    lists = np.full((1, 50), -1, dtype=np.int64)
    lists[0, :33] = np.arange(5, 170, 5)[:33]
    unnamed = torch.tensor([p for p in range(200) if p not in lists[0]], device=device)
    flat_k[rows[unnamed]] = math.nan
    flat_v[rows[unnamed]] = math.inf
    out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2],
                                        torch.from_numpy(lists).to(device), return_lse=True)
    c.check(out, lse, 128**-0.5, lists=lists)


def test_selected_lists_of_every_key_equal_attention(device) -> None:
    c = Case(device, 4, [777, 1000], [1, 1], 16, 4, 128, 32, BF16)
    table, lengths, _ = c.device_args()
    q = c.q.to(device)
    every = torch.arange(1000, device=device).expand(2, 1000)
    out, lse = paged.selected_attention(q, c.cache, table, lengths, every.to(torch.int32), return_lse=True)
    c.check(out, lse, 128**-0.5)
    empty, lse = paged.selected_attention(q, c.cache, table, lengths, every[:, :0], return_lse=True)
    assert (empty == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("selected", [False, True])
def test_offsets_past_32_bits(device, selected) -> None:
    """Pages beyond 4 GiB of keys."""

    dim, page, kv_heads = 128, 64, 8
    pages = (5 << 30) // (page * kv_heads * dim * 2)
    keys = torch.zeros(pages, page, kv_heads, dim, dtype=BF16, device=device)
    values = torch.zeros_like(keys)
    cache = paged.PagedCache(keys, values)
    gen = torch.Generator().manual_seed(6)
    n = 150
    table = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device=device)
    k, v = (torch.randn(n, kv_heads, dim, generator=gen).to(BF16).to(device) for _ in range(2))
    rows = paged.cache_rows(cache, table, torch.arange(n, device=device), torch.zeros(n, dtype=torch.int64, device=device))
    paged.append(cache, k, v, rows, torch.zeros(n, dtype=torch.int64, device=device))
    q = torch.randn(1, 16, dim, generator=gen).to(BF16)
    lengths = torch.tensor([n], dtype=torch.int32, device=device)
    if selected:
        out = paged.selected_attention(q.to(device), cache, table, lengths, torch.arange(n, device=device)[None])
    else:
        out = paged.attention(q.to(device), cache, table, lengths)
    k64, v64 = _f64(k), _f64(v)
    for h in range(16):
        ref, _, weighted, _ = oracle.attend(_f64(q)[0, h], k64[:, h // 2], v64[:, h // 2], dim**-0.5)
        assert (np.abs(_f64(out)[0, h] - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-7.9 * weighted + 1e-9).all()


def test_attention_reads_strided_queries_and_a_side_stream(device) -> None:
    c = Case(device, 8, [100, 260], [1, 1], 8, 2, 128, 16, BF16)
    wide = torch.zeros(2, 8 * 128 + 512, dtype=BF16, device=device)
    table, lengths, starts = c.device_args()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        wide[:, 256:256 + 1024] = c.q.reshape(2, -1).to(device)
        out, lse = paged.attention(wide[:, 256:256 + 1024].view(2, 8, 128), c.cache, table, lengths, starts, return_lse=True)
    side.synchronize()
    c.check(out, lse, 128**-0.5)


def test_decode_step_in_a_graph(device) -> None:
    """append, attention and selected attention captured together; every replay
    equals the eager step on the same inputs, the cache growing between them."""

    batch, heads, kv_heads, dim, page = 3, 8, 2, 128, 16
    gen = torch.Generator().manual_seed(12)
    cache = paged.new_cache(64, page, kv_heads, dim, device=device)
    eager = paged.new_cache(64, page, kv_heads, dim, device=device)
    for c in (cache, eager):
        c.keys.copy_(torch.randn(c.keys.shape, generator=torch.Generator().manual_seed(1)))
        c.values.copy_(torch.randn(c.values.shape, generator=torch.Generator().manual_seed(2)))
    table = torch.randperm(64, generator=gen)[:60].view(3, 20).to(torch.int32).to(device)
    lengths = torch.tensor([100, 33, 250], dtype=torch.int32, device=device)
    qkv = [torch.randn(batch, n, dim, generator=gen).to(BF16).to(device) for n in (heads, kv_heads, kv_heads)]
    lists = torch.zeros(batch, 24, dtype=torch.int64, device=device)
    rows = torch.full((batch,), -1, dtype=torch.int64, device=device)
    positions = torch.zeros(batch, dtype=torch.int64, device=device)

    def step(c):
        q = paged.append(c, qkv[1], qkv[2], rows, positions, queries=qkv[0])
        return paged.attention(q, c, table, lengths), paged.selected_attention(q, c, table, lengths, lists)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(cache)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step(cache)
    for _ in range(4):
        lengths += 1
        positions.copy_(lengths.long() - 1)
        rows.copy_(paged.cache_rows(cache, table, positions))
        lists.copy_(torch.randint(0, 33, lists.shape, generator=gen))
        for x in qkv:
            x.copy_(torch.randn(x.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        for got, ref in zip(captured, want):
            assert torch.equal(got, ref)
    assert torch.equal(cache.keys, eager.keys) and torch.equal(cache.values, eager.values)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rope_dim,page,dtype,layout", [
    (1, 32, 8, 128, 128, 64, BF16, "nhd"),
    (7, 0, 3, 64, 64, 16, F16, "hnd"),
    (33, 5, 1, 128, 64, 1, BF16, "wide"),
    (19, 6, 2, 256, 256, 32, FP8, "nhd"),
    (40, 0, 4, 64, 32, 8, FP8, "hnd"),
    (5, 8, 8, 256, 0, 16, F16, "wide"),
    (11, 70, 1, 128, 16, 16, BF16, "nhd"),   # more heads than one workgroup's units
])
def test_append(device, tokens, heads, kv_heads, dim, rope_dim, page, dtype, layout) -> None:
    print(f"append {tokens} {heads}/{kv_heads}x{dim} rope {rope_dim} page {page} {dtype} {layout}", flush=True)
    row = BF16 if dtype == FP8 else dtype
    c = Case(device, tokens, [page], [1], kv_heads, kv_heads, dim, page, dtype, layout=layout, spare=tokens // page + 3)
    gen = torch.Generator().manual_seed(tokens)
    k, v = (torch.randn(tokens, kv_heads, dim, generator=gen).to(row) for _ in range(2))
    k[0, 0] = 0  # a head of zeros keeps the least scale
    if tokens > 2:
        v[2, 0, 3] = 300.0
    q = torch.randn(tokens, heads, dim, generator=gen).to(row) if heads else None
    rows = torch.randperm(c.cache.rows, generator=gen)[:tokens]
    if tokens > 4:
        rows[3], rows[4] = -1, c.cache.rows
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen)
    before = [_f64(x) for x in (c.cache.keys, c.cache.values)]
    scales = [None if s is None else s.clone().cpu().numpy() for s in (c.cache.key_scales, c.cache.value_scales)]
    store = torch.zeros(tokens, 2, kv_heads, dim, dtype=row)  # keys and values as slices of one projection
    store[:, 0], store[:, 1] = k, v
    store = store.to(device)
    got = paged.append(c.cache, store[:, 0], store[:, 1], rows.to(device), positions.to(device),
                       queries=None if q is None else q.to(device), rope_dim=rope_dim, theta=5000.0)
    u = UNIT[row]
    turned = {0: oracle.rotate(_f64(k), positions.numpy(), rope_dim, 5000.0), 1: _f64(v)}
    after = [_f64(x) for x in (c.cache.keys, c.cache.values)]
    for which in (0, 1):
        want, new = before[which].reshape(-1, kv_heads, dim), after[which].reshape(-1, kv_heads, dim)
        live = [t for t in range(tokens) if 0 <= rows[t] < c.cache.rows]
        x = turned[which][live]
        at = rows[live].numpy()
        pair = _f64(k if which == 0 else v)[live]
        size = np.abs(pair).max(axis=-1, keepdims=True) * (2.0 if which == 0 else 0.0)
        slack = 2.0**-20 * size  # fp32 angle, products and sums
        if dtype == FP8:
            s = (c.cache.key_scales, c.cache.value_scales)[which].cpu().numpy().reshape(-1, kv_heads)
            expected = oracle.head_scale(x)
            assert (np.abs(s[at] - expected) <= 2.0**-23 * expected + slack[..., 0] / 448).all()
            keep = np.ones(c.cache.rows, bool)
            keep[at] = False
            assert np.array_equal(s[keep], scales[which].reshape(-1, kv_heads)[keep])
            # e4m3: half an ulp is 2^-4 of a normal value, 2^-10 below 2^-6
            near = np.abs(new[at] * s[at][..., None].astype(np.float64) - x)
            assert (near <= 2.0**-4 * np.abs(x) + 2.0**-10 * s[at][..., None] + slack).all()
        else:
            bound = u * np.abs(x) + slack if which == 0 else 0.0
            assert (np.abs(new[at] - x) <= bound).all()
        others = np.setdiff1d(np.arange(c.cache.rows), at)
        assert np.array_equal(new[others], want[others], equal_nan=True)
    if q is None:
        assert got is None
    else:
        ref = oracle.rotate(_f64(q), positions.numpy(), rope_dim, 5000.0)
        size = 2 * np.abs(_f64(q)).max(axis=-1, keepdims=True)
        assert got.dtype == row
        assert (np.abs(_f64(got) - ref) <= u * np.abs(ref) + 2.0**-20 * size).all()


def test_append_of_no_tokens(device) -> None:
    cache = paged.new_cache(2, 16, 2, 64, device=device)
    none = torch.zeros(0, 2, 64, dtype=BF16, device=device)
    at = torch.zeros(0, dtype=torch.int64, device=device)
    assert paged.append(cache, none, none, at, at) is None
    table = torch.zeros(1, 2, dtype=torch.int32, device=device)
    lengths = torch.zeros(1, dtype=torch.int32, device=device)
    assert paged.attention(none, cache, table, lengths).shape == (0, 2, 64)
    out, lse = paged.selected_attention(none, cache, table, lengths, torch.zeros(0, 8, dtype=torch.int64, device=device),
                                        return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


def test_indexer_selection_feeds_the_attention(device) -> None:
    """A decode step whole: the indexer's top-k of its keys names the positions
    that the attention reads, and k at the context's length equals the dense
    attention."""

    batch, n, heads, kv_heads, dim = 2, 600, 8, 2, 128
    c = Case(device, 21, [n, n], [1, 1], heads, kv_heads, dim, 32, BF16)
    gen = torch.Generator().manual_seed(3)
    iq = torch.randn(batch, 64, 128, generator=gen).to(BF16).to(device)
    iw = torch.randn(batch, 64, generator=gen).to(device)
    ik = torch.randn(batch, n, 128, generator=gen).to(BF16).to(device)
    for k in (100, n, 700):
        idx = decode.indexer_topk(iq, iw, ik, k)
        out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2], idx, return_lse=True)
        c.check(out, lse, dim**-0.5, lists=idx.cpu().numpy())


def test_refusals(device) -> None:
    cache = paged.new_cache(4, 16, 2, 128, device=device)
    table = torch.zeros(2, 2, dtype=torch.int32, device=device)
    lengths = torch.ones(2, dtype=torch.int32, device=device)
    q = torch.zeros(2, 4, 128, dtype=BF16, device=device)
    kv = torch.zeros(2, 2, 128, dtype=BF16, device=device)
    at = torch.zeros(2, dtype=torch.int64, device=device)

    def refuses(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    refuses("page_size", paged.new_cache, 4, 12, 2, 128, device=device)
    refuses("head_dim", paged.new_cache, 4, 16, 2, 96, device=device)
    refuses("BF16, FP16 or FP8", paged.new_cache, 4, 16, 2, 128, dtype=torch.float32, device=device)
    refuses("aligned", paged.PagedCache, cache.keys.transpose(1, 3).contiguous().transpose(1, 3), cache.values)
    fp8 = cache.keys.to(FP8)
    refuses("scales", paged.PagedCache, fp8, fp8)
    refuses("only an fp8", paged.PagedCache, cache.keys, cache.values, torch.zeros(4, 16, 2, device=device))
    refuses("both be", paged.append, cache, kv[:, :1], kv[:, :1], at, at)
    refuses("dtype", paged.append, cache, kv.half(), kv.half(), at, at)
    refuses(r"\[tokens\]", paged.append, cache, kv, kv, at[:1], at)
    refuses("integers", paged.append, cache, kv, kv, at.float(), at)
    refuses("rope_dim", paged.append, cache, kv, kv, at, at, rope_dim=24)
    refuses("rope_dim", paged.append, cache, kv, kv, at, at, rope_dim=144)
    refuses("theta", paged.append, cache, kv, kv, at, at, theta=0.0)
    refuses("queries", paged.append, cache, kv, kv, at, at, queries=q[:1])
    refuses("head_dim", paged.attention, q[..., :64], cache, table, lengths)
    refuses("multiple", paged.attention, q[:, :3], cache, table, lengths)
    refuses("dtype", paged.attention, q.half(), cache, table, lengths)
    refuses("one GPU", paged.attention, q.cpu(), cache, table, lengths)
    refuses("page_table", paged.attention, q, cache, table[0], lengths)
    refuses("lengths", paged.attention, q, cache, table, lengths[:1])
    refuses("starts", paged.attention, q, cache, table, lengths, lengths)
    refuses("same number", paged.attention, q[:1], cache, table, lengths)
    refuses("indices", paged.selected_attention, q, cache, table, lengths, at)
    refuses("integers", paged.selected_attention, q, cache, table, lengths, at.float()[:, None])
