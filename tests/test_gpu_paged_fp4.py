"""The 4-bit paged cache against float64: append (codes and powers to the bit), reading
back, and attention of one token, a chunk, a prompt and selected keys.

An fp4 cache stands for values that bf16 holds exactly, so the attention's bounds are
those of a bf16 cache of the same values (``test_gpu_paged``)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import paged
from oracle import paged as oracle
from test_gpu_paged import BF16, F16, FP8, Case, _f64

pytestmark = pytest.mark.gpu

FP4 = torch.float4_e2m1fn_x2
E8M0 = torch.float8_e8m0fnu


def _bytes(x: torch.Tensor) -> np.ndarray:
    return x.view(torch.uint8).cpu().numpy()


class Case4(Case):
    """A case of ``test_gpu_paged`` over a 4-bit cache: random codes under random
    powers of two, those of stale rows NaN."""

    def __init__(self, device, seed, lengths, chunks, heads, kv_heads, dim, page, *, layout="paged", **kw):
        super().__init__(device, seed, lengths, chunks, heads, kv_heads, dim, page, BF16, **kw)
        pages = self.cache.pages
        stale = torch.isnan(self.cache.keys[:, :, 0, 0]).cpu()
        parts = []
        for name in ("keys64", "values64"):
            codes = torch.randint(0, 256, (pages, page, kv_heads, dim // 2), generator=self.gen, dtype=torch.uint8)
            powers = torch.randint(122, 128, (pages, kv_heads, page, dim // 32), generator=self.gen, dtype=torch.uint8)
            powers[stale[:, None].expand(-1, kv_heads, -1)] = 255
            setattr(self, name, oracle.fp4_values(codes.numpy(), powers.transpose(1, 2).numpy()))
            if layout == "paged":  # head by head within a page
                codes = codes.transpose(1, 2).contiguous().to(device).transpose(1, 2)
            elif layout == "wide":  # beside other bytes
                store = torch.zeros(pages, page, kv_heads, dim, dtype=torch.uint8, device=device)
                store[..., dim // 2:] = codes.to(device)
                codes = store[..., dim // 2:]
            else:
                codes = codes.to(device)
            parts.append((codes.view(FP4), powers.to(device).view(E8M0)))
        (keys, key_powers), (values, value_powers) = parts
        self.cache = paged.PagedCache(keys, values, key_powers, value_powers)
        self.written = ~stale


ATTENTION = [
    # lengths, chunks, heads, kv_heads, dim, page, layout
    ([1], [1], 1, 1, 64, 1, "paged"),
    ([1, 2, 31, 32, 33], [1] * 5, 4, 2, 128, 16, "paged"),
    ([129, 0, 700], [1, 1, 1], 8, 2, 128, 64, "rows"),
    ([300, 77], [1, 1], 8, 8, 64, 32, "wide"),
    ([513, 64], [1, 1], 6, 1, 256, 16, "wide"),
    ([211, 33], [1, 1], 16, 2, 256, 8, "paged"),
    ([95, 130], [1, 1], 40, 1, 128, 4, "rows"),      # 40 heads of one kv head: three row tiles
    ([40, 70, 9], [5, 0, 9], 7, 1, 64, 16, "paged"),  # an odd group, an empty chunk, a whole sequence
    ([3, 50], [6, 2], 4, 4, 128, 16, "paged"),       # more new tokens than keys: early rows see nothing
    ([0, 0], [2, 3], 4, 2, 64, 16, "paged"),         # nothing cached at all
    ([260], [130], 6, 2, 128, 16, "paged"),          # a chunk of several row tiles
    ([200, 517, 90], [200, 33, 1], 8, 2, 128, 32, "rows"),
    ([150], [150], 4, 2, 64, 1, "paged"),
    ([700, 515], [50, 50], 8, 2, 64, 16, "wide"),
    ([170, 301], [64, 129], 5, 1, 256, 64, "paged"),
    ([140], [70], 12, 2, 256, 16, "rows"),
    ([2100], [3], 4, 4, 128, 256, "paged"),          # pieces of one sequence
    ([1100], [1000], 16, 1, 128, 16, "paged"),
    ([1900], [40], 16, 1, 64, 16, "paged"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,layout", ATTENTION)
def test_attention(device, lengths, chunks, heads, kv_heads, dim, page, layout, causal) -> None:
    print(f"fp4 attention {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} {layout} {causal}", flush=True)
    c = Case4(device, 5 + dim, lengths, chunks, heads, kv_heads, dim, page, layout=layout)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), causal=causal, return_lse=True)
    c.check(out, lse, dim**-0.5, causal=causal)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
def test_decode_longer_than_one_lookup(device, dim, page) -> None:
    """Pieces of more than 2048 keys, many heads."""

    c = Case4(device, 3, [5003, 2049, 4096], [1, 1, 1], 400, 400, dim, page)
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(starts=False), scale=0.3, return_lse=True)
    keep = slice(0, 400, 57)
    c.q, c.heads = c.q[:, keep], len(range(0, 400, 57))
    c.keys64, c.values64 = c.keys64[:, :, keep], c.values64[:, :, keep]
    c.check(out[:, keep], lse[:, keep], 0.3)


@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,page,k", [
    ([1], [1], 1, 1, 64, 1, 1),
    ([300, 40], [1, 1], 8, 2, 128, 16, 64),
    ([300, 4000, 0], [1, 1, 1], 8, 2, 128, 64, 257),
    ([500, 90], [1, 1], 32, 1, 64, 32, 100),       # two row tiles of one token's heads
    ([90, 33, 7], [40, 0, 7], 6, 2, 256, 16, 30),
    ([400], [9], 12, 4, 256, 8, 333),
    ([5000], [1], 4, 4, 128, 16, 4500),
    ([700], [600], 4, 4, 64, 16, 100),             # a list to a wave
])
def test_selected(device, lengths, chunks, heads, kv_heads, dim, page, k) -> None:
    print(f"fp4 selected {lengths} {chunks} {heads}/{kv_heads}x{dim} page {page} k {k}", flush=True)
    c = Case4(device, 11 + k, lengths, chunks, heads, kv_heads, dim, page)
    tokens = sum(chunks)
    lists = np.full((tokens, k), -1, dtype=np.int64)
    rng = np.random.default_rng(k)
    for b, n in enumerate(lengths):
        for t in range(c.starts[b], c.starts[b + 1]):
            m = min(n, int(rng.integers(0, k + 1)) if t % 3 else k)
            lists[t, rng.permutation(k)[:m]] = rng.permutation(n)[:m]
            junk = np.flatnonzero(lists[t] < 0)[::2]
            lists[t, junk] = rng.choice([-1, -5, n, n + 1000000, 2**40, -2**62], len(junk))
    if tokens > 1:
        lists[-1] = -1
    out, lse = paged.selected_attention(c.q.to(device), c.cache, *c.device_args()[:2], torch.from_numpy(lists).to(device),
                                        c.device_args()[2], return_lse=True)
    c.check(out, lse, dim**-0.5, lists=lists)


@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim", [
    ([90], [3], 4, 2, 128), ([200, 40], [30, 30], 8, 2, 64), ([333], [200], 8, 2, 128), ([150], [40], 4, 1, 256),
    ([2500], [2], 4, 4, 64),
])
def test_nan_reaches_the_rows_that_see_it_alone(device, lengths, chunks, heads, kv_heads, dim) -> None:
    """A later token's block without a value is NaN in its dims of the outputs that see
    it; a key's is NaN in every dim of those."""

    for which in ("keys", "values"):
        c = Case4(device, 31, lengths, chunks, heads, kv_heads, dim, 16)
        want, want_lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
        n, new = lengths[0], chunks[0]
        at = n - new + new // 2  # seen by the last new tokens of the first sequence
        row = int(paged.cache_rows(c.cache, c.table.to(device), torch.tensor([at], device=device),
                                   torch.zeros(1, dtype=torch.int64, device=device)))
        powers = (c.cache.key_scales if which == "keys" else c.cache.value_scales).view(torch.uint8)
        powers[row // 16, kv_heads - 1, row % 16, 1] = 255
        got, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
        hit = torch.zeros(got.shape, dtype=torch.bool, device=device)
        heads_of = slice((kv_heads - 1) * (heads // kv_heads), heads)
        hit[new // 2:new, heads_of, slice(None) if which == "keys" else slice(32, 64)] = True
        assert torch.isnan(got[hit]).all()
        assert torch.equal(got[~hit], want[~hit])
        assert torch.equal(torch.isnan(lse), hit.all(-1)) and torch.equal(lse[~hit.all(-1)], want_lse[~hit.all(-1)])


def test_first_scores_far_apart(device) -> None:
    """Scores that rise and fall by powers of two over the keys."""

    c = Case4(device, 8, [700, 300], [40, 1], 8, 2, 128, 16)
    for scale in (30.0, 1e-3):
        out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), scale=scale, return_lse=True)
        c.check(out, lse, scale)


APPEND = [
    # tokens, heads, kv_heads, dim, rope_dim, page, layout
    (1, 32, 8, 128, 128, 64, "paged"),
    (7, 0, 3, 64, 64, 16, "paged"),
    (33, 5, 1, 128, 64, 1, "rows"),
    (19, 6, 2, 256, 256, 32, "wide"),
    (40, 0, 4, 64, 32, 8, "paged"),
    (5, 8, 8, 256, 0, 16, "paged"),
    (11, 70, 1, 128, 16, 16, "rows"),    # more heads than one workgroup's units; runs of 8 turned with runs far off
    (13, 2, 2, 128, 48, 16, "paged"),    # half of the rotated dims is no whole block
    (300, 0, 2, 64, 64, 16, "paged"),
]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rope_dim,page,layout", APPEND)
def test_append(device, tokens, heads, kv_heads, dim, rope_dim, page, layout) -> None:
    """Every power and value is that of the float64 oracle: rotated in 64 bits, a key
    is rounded once.  (The angle, up to 2^20, is itself off by 2^-33: a key that lies
    within 1e-9 of a border between two codes may go either way.)"""

    print(f"fp4 append {tokens} {heads}/{kv_heads}x{dim} rope {rope_dim} page {page} {layout}", flush=True)
    c = Case4(device, tokens, [page], [1], kv_heads, kv_heads, dim, page, layout=layout, spare=tokens // page + 3)
    gen = torch.Generator().manual_seed(tokens)
    k, v = (torch.randn(tokens, kv_heads, dim, generator=gen).to(BF16) for _ in range(2))
    k *= torch.exp2(torch.randint(-20, 20, (tokens, kv_heads, 1), generator=gen)).to(BF16)
    v[0, 0] = 0                       # blocks of zeros have the least power
    v[-1, -1, 3], v[-1, -1, 40] = 3e38, 1e-39
    if tokens > 2:
        v[1, 0, 33], v[2, 0, 5] = math.nan, -math.inf
        # every border between two codes, and the values next to them, in blocks of power 1
        grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0])
        near = torch.cat([grid, grid * (1 + 2.0**-7), grid * (1 - 2.0**-8)])
        for t in range(3, min(tokens, 5)):
            v[t, 0, :30] = (near if t == 3 else -near).to(BF16)
            v[t, 0, 30:32] = 7.0
    q = torch.randn(tokens, heads, dim, generator=gen).to(BF16) if heads else None
    rows = torch.randperm(c.cache.rows, generator=gen)[:tokens]
    if tokens > 6:
        rows[5], rows[6] = -1, c.cache.rows
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen)
    before = [_bytes(x).copy() for x in (c.cache.keys, c.cache.values, c.cache.key_scales, c.cache.value_scales)]
    store = torch.zeros(tokens, 2, kv_heads, dim, dtype=BF16)  # keys and values as slices of one projection
    store[:, 0], store[:, 1] = k, v
    store = store.to(device)
    got = paged.append(c.cache, store[:, 0], store[:, 1], rows.to(device), positions.to(device),
                       queries=None if q is None else q.to(device), rope_dim=rope_dim, theta=5000.0)
    live = [t for t in range(tokens) if 0 <= rows[t] < c.cache.rows]
    at = rows[live].numpy()
    others = np.setdiff1d(np.arange(c.cache.rows), at)
    read = paged.read(c.cache, rows[live].to(device))
    turned = (oracle.rotate(_f64(k), positions.numpy(), rope_dim, 5000.0), _f64(v))
    for which, (codes, powers) in enumerate(((c.cache.keys, c.cache.key_scales), (c.cache.values, c.cache.value_scales))):
        want, want_powers = oracle.fp4(turned[which][live])
        codes, powers = _bytes(codes), _bytes(powers).transpose(0, 2, 1, 3)
        flat = codes.reshape(-1, kv_heads, dim // 2)
        assert np.array_equal(powers.reshape(-1, kv_heads, dim // 32)[at], want_powers)
        assert np.array_equal(oracle.fp4_values(flat[at], want_powers), want, equal_nan=True)
        assert np.array_equal(flat[others], before[which].reshape(-1, kv_heads, dim // 2)[others])
        old = before[2 + which].transpose(0, 2, 1, 3).reshape(-1, kv_heads, dim // 32)
        assert np.array_equal(powers.reshape(-1, kv_heads, dim // 32)[others], old[others])
        assert read[which].dtype == BF16 and np.array_equal(_f64(read[which]), want, equal_nan=True)
    if q is None:
        assert got is None
    else:
        ref = oracle.rotate(_f64(q), positions.numpy(), rope_dim, 5000.0)
        size = 2 * np.abs(_f64(q)).max(axis=-1, keepdims=True)
        assert got.dtype == BF16 and (np.abs(_f64(got) - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-20 * size).all()


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "wide"])
def test_read_of_other_caches(device, dtype, layout) -> None:
    c = Case(device, 17, [70, 33], [1, 1], 6, 3, 64, 16, dtype, layout=layout)
    rows = torch.tensor([5, -1, 0, c.cache.rows - 1, c.cache.rows, 5, 1 << 40, 40], device=device)
    keys, values = paged.read(c.cache, rows)
    inside = ((rows >= 0) & (rows < c.cache.rows)).cpu().numpy()
    for got, cached, scales in ((keys, c.cache.keys, c.cache.key_scales), (values, c.cache.values, c.cache.value_scales)):
        want = _f64(cached)
        if scales is not None:
            want = want * scales.double().cpu().numpy()[..., None]
        want = want.reshape(-1, 3, 64)[rows.cpu().numpy()[inside]]
        out = _f64(got)
        assert (out[~inside] == 0).all()
        if dtype == FP8:
            fine = np.isfinite(want)
            assert np.array_equal(np.isnan(out[inside]), ~fine)
            assert (np.abs(out[inside] - want)[fine] <= 2.0**-8 * np.abs(want)[fine] + 2.0**-24 * np.abs(want)[fine]).all()
        else:
            assert np.array_equal(out[inside], want, equal_nan=True)
    none, _ = paged.read(c.cache, rows[:0])
    assert none.shape == (0, 3, 64)


def test_read_and_append_past_32_bits(device) -> None:
    """Codes beyond 4 GiB of a cache, powers beyond 256 MiB."""

    page, kv_heads, dim = 64, 8, 256
    pages = (5 << 30) // (page * kv_heads * dim // 2)
    cache = paged.new_cache(pages, page, kv_heads, dim, dtype=FP4, device=device)
    gen = torch.Generator().manual_seed(6)
    k, v = (torch.randn(5, kv_heads, dim, generator=gen).to(BF16) for _ in range(2))
    rows = torch.tensor([cache.rows - 1, 0, cache.rows // 2, cache.rows - 64, 65])
    positions = torch.arange(5)
    paged.append(cache, k.to(device), v.to(device), rows.to(device), positions.to(device), rope_dim=0)
    for got, x in zip(paged.read(cache, rows.to(device)), (k, v)):
        assert np.array_equal(_f64(got), oracle.fp4(_f64(x))[0])
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=device)
    paged.append(cache, k[:1].expand(64, -1, -1).to(device), v[:1].expand(64, -1, -1).to(device),
                 torch.arange(cache.rows - 64, cache.rows, device=device), torch.zeros(64, device=device).long(), rope_dim=0)
    q = torch.randn(1, 16, dim, generator=gen).to(BF16).to(device)
    out = paged.attention(q, cache, table, torch.tensor([64], dtype=torch.int32, device=device))
    want = oracle.fp4(_f64(v))[0][0].repeat(2, axis=0)  # 64 keys alike
    assert (np.abs(_f64(out)[0] - want) <= 2.0**-7 * np.abs(want)).all()


def test_decode_in_a_graph(device) -> None:
    """append, both attentions and read captured together; every replay equals the
    eager step on the same inputs, the cache growing between them."""

    batch, heads, kv_heads, dim, page = 3, 8, 2, 128, 16
    gen = torch.Generator().manual_seed(12)
    caches = [paged.new_cache(64, page, kv_heads, dim, dtype=FP4, device=device) for _ in range(2)]
    fill = [torch.randn(1024, kv_heads, dim, generator=gen).to(BF16).to(device) for _ in range(2)]
    every = torch.arange(1024, device=device)
    for c in caches:
        paged.append(c, *fill, every, every)
    table = torch.randperm(64, generator=gen)[:60].view(3, 20).to(torch.int32).to(device)
    lengths = torch.tensor([100, 33, 250], dtype=torch.int32, device=device)
    qkv = [torch.randn(batch, n, dim, generator=gen).to(BF16).to(device) for n in (heads, kv_heads, kv_heads)]
    lists = torch.zeros(batch, 24, dtype=torch.int64, device=device)
    rows = torch.full((batch,), -1, dtype=torch.int64, device=device)
    positions = torch.zeros(batch, dtype=torch.int64, device=device)

    def step(c):
        q = paged.append(c, qkv[1], qkv[2], rows, positions, queries=qkv[0])
        return (paged.attention(q, c, table, lengths), paged.selected_attention(q, c, table, lengths, lists),
                *paged.read(c, rows))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(caches[0])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step(caches[0])
    for _ in range(4):
        lengths += 1
        positions.copy_(lengths.long() - 1)
        rows.copy_(paged.cache_rows(caches[0], table, positions))
        lists.copy_(torch.randint(0, 33, lists.shape, generator=gen))
        for x in qkv:
            x.copy_(torch.randn(x.shape, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(captured, step(caches[1])):
            assert torch.equal(got, ref)
    for x, y in zip(paged.read(caches[0], every), paged.read(caches[1], every)):
        assert torch.equal(x, y)


def test_refusals(device) -> None:
    cache = paged.new_cache(4, 16, 2, 128, dtype=FP4, device=device)
    assert (cache.head_dim, cache.row_dtype, cache.rows) == (128, BF16, 64)

    def refuses(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    k, v, ks, vs = cache.keys, cache.values, cache.key_scales, cache.value_scales
    refuses("scales", paged.PagedCache, k, v)
    refuses("scales", paged.PagedCache, k, v, ks)
    refuses("scales", paged.PagedCache, k, v, ks.view(torch.uint8), vs)
    refuses("scales", paged.PagedCache, k, v, ks.transpose(1, 2), vs)
    refuses("scales", paged.PagedCache, k, v, ks[..., :2].contiguous(), vs)
    refuses("head_dim", paged.new_cache, 4, 16, 2, 32, dtype=FP4, device=device)
    refuses("head_dim", paged.new_cache, 4, 16, 2, 96, dtype=FP4, device=device)
    refuses("page_size", paged.new_cache, 4, 12, 2, 128, dtype=FP4, device=device)
    kv = torch.zeros(2, 2, 128, dtype=F16, device=device)
    at = torch.zeros(2, dtype=torch.int64, device=device)
    refuses("FP4", paged.append, cache, kv, kv, at, at)
    refuses("FP4", paged.attention, kv, cache, at[:1, None].int(), at[:1].int())
    refuses(r"rows must be \[n\]", paged.read, cache, at[None])
    refuses("integers", paged.read, cache, at.float())
