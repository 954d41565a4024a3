"""The split of attention over workgroups, restated: for any batch, padded or not,
every row tile's keys are dealt to pieces once, the pieces fit the launch, their
partial results the workspace that the library asks for, and their counters the
workspace's first 16 KiB."""

from __future__ import annotations

import ctypes
import random

import pytest

from dsa_amd import _lib

STREAM_ROWS, LEAST_KEYS, COUNTERS, MOST_SPLITS = 16, 256, 4096, 256
RESIDENT = {64: 768, 128: 512, 256: 256}


def _up(a: int, b: int) -> int:
    return -(-a // b)


def _plan(dim, element, kv_heads, page, sequences, tokens, heads, columns, uniform):
    """Launches as dicts, and the parts and rows of the workspace."""

    group, capacity = heads // kv_heads, columns * page
    uniform = uniform or sequences == 1
    each = tokens // sequences * group
    few = not uniform and tokens <= sequences
    launches, parts, rows = [], 0, 0

    def at_most(tiles, cuts):
        return min(tiles * _up(capacity, LEAST_KEYS), tiles + cuts)

    if not uniform or each <= STREAM_ROWS:
        beside = dim * element == 128 and kv_heads % 2 == 0 and sequences * capacity * kv_heads >= 1 << 19
        kinds = kv_heads // 2 if beside else kv_heads
        cuts = _up(256 if beside else RESIDENT[dim], kinds)
        tiles = min(tokens, sequences) + (tokens * group // STREAM_ROWS if few else 0)
        held = each if uniform else STREAM_ROWS
        launches.append(dict(tile=16, unit=32, cuts=cuts, whole=0, least=1, most=1 << 40 if few else STREAM_ROWS,
                             grid=_up(at_most(tiles, cuts), 8) * 8, rows=held, kinds=kinds, counts=True))
        parts = 2 * cuts * kv_heads * held
    if each > STREAM_ROWS if uniform else not few:
        prefill = dim == 256 or tokens * group > 128 * sequences
        size = (128 if dim == 256 else 256) if prefill else 128
        cuts = _up(256 if prefill else RESIDENT[dim], kv_heads)
        if uniform:
            tiles = sequences * _up(tokens // sequences * group, size)
        else:
            tiles = (tokens * group + (size - 1) * min(tokens, sequences)) // size
        rest = tiles % cuts
        alone = sequences == 1 and tiles >= cuts
        cut = rest > 0 and tiles < 8 * cuts and (tiles < 2 * cuts or 8 * tokens <= 5 * capacity) if alone else tiles < 2 * cuts
        launch = dict(tile=size, unit=64, cuts=0, whole=0, least=STREAM_ROWS + 1 if launches else 1, most=1 << 40,
                      grid=tiles, rows=size, kinds=kv_heads, counts=False)
        if cut:
            launch["cuts"] = cuts
            if alone:
                launch.update(whole=tiles - rest, grid=tiles - rest + max(cuts, rest))
            else:
                launch["grid"] = at_most(tiles, cuts)
            rows = tokens * heads
            parts = max(parts, 2 * cuts * kv_heads * size)
        launches.append(launch)
    return launches, parts, rows


def _pieces(launch, group, spans, keys):
    """Every piece that the launch's workgroups find: sequence, tile, first unit, units, slot and pieces of its tile."""

    least = LEAST_KEYS // launch["unit"]
    tiles, units = [], []
    for n, k in zip(spans, keys):
        rows = n * group
        t = _up(rows, launch["tile"]) if launch["least"] <= rows <= launch["most"] else 0
        tiles.append(t)
        units.append(_up(k, launch["unit"]) if t or launch["whole"] else 0)
    if launch["whole"]:
        found = [(0, t, 0, max(1, units[0]), 0, 1) for t in range(min(tiles[0], launch["whole"]))]
        rest = tiles[0] - launch["whole"]
        if rest > 0:
            count = min(max(1, min(launch["cuts"] // rest, units[0] // least)), MOST_SPLITS)
            long = max(1, _up(units[0], count))
            found += [(0, launch["whole"] + t, i * long, long, t * count, count) for t in range(rest) for i in range(count)]
        return found
    length = 0x7FFFFFFF
    if launch["cuts"]:
        work = sum(t * u for t, u in zip(tiles, units))
        length = max(least, _up(max(units), MOST_SPLITS), _up(work, launch["cuts"]))
        if len(spans) <= 64:
            for _ in range(8):
                if sum(t * max(1, _up(u, length)) for t, u in zip(tiles, units)) <= launch["cuts"]:
                    break
                length += _up(length, 32)
    found, slot = [], 0
    for b, (t, u) in enumerate(zip(tiles, units)):
        count = max(1, _up(u, length))
        long = max(1, _up(u, count))
        for tile in range(t):
            found += [(b, tile, i * long, long, slot + tile * count, count) for i in range(count)]
        slot += t * count if count > 1 else 0
    return found


def _draw(rng: random.Random) -> dict:
    def spread(low, high):
        return min(high, int(low * (high / low) ** rng.random() + 0.5))

    dim, element = rng.choice([64, 128, 256]), rng.choice([1, 2])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16, 64, 200, 1024])
    group = rng.choice([1, 2, 4, 7, 8, 16, 40])
    sequences = spread(1, rng.choice([1, 8, 64, 300]))
    page, columns = rng.choice([1, 16, 64, 256]), spread(1, 600)
    most = rng.choice([1, 1, 3, 40, 700])
    keys = [rng.randint(0, columns * page) if rng.random() < 0.9 else 0 for _ in range(sequences)]
    uniform = rng.random() < 0.4
    if uniform:
        spans = [spread(1, most)] * sequences
    else:
        spans = [rng.choice([0, 1, spread(1, most)]) for _ in range(sequences)]
    tokens = sum(spans)
    if not uniform:
        tokens += rng.choice([0, 0, 1, spread(1, 800)])  # padding
        if tokens == 0:
            tokens = 1
    return dict(dim=dim, element=element, kv_heads=kv_heads, heads=kv_heads * group, page=page, columns=columns,
                sequences=sequences, tokens=tokens, spans=spans, keys=keys, uniform=uniform)


@pytest.mark.parametrize("seed", range(8))
def test_pieces_fit(seed) -> None:
    rng = random.Random(seed)
    lib = _lib.load()
    for _ in range(400):
        c = _draw(rng)
        launches, parts, rows = _plan(c["dim"], c["element"], c["kv_heads"], c["page"], c["sequences"], c["tokens"],
                                      c["heads"], c["columns"], c["uniform"])
        stride = c["kv_heads"] * c["dim"]
        cache = _lib.PagedCacheC(256, 256, 256, 256, 8, c["page"] * stride, stride, c["dim"], c["page"] * stride, stride,
                                 c["dim"], c["page"], c["kv_heads"], c["dim"],
                                 _lib.DTYPE_FP8_E4M3 if c["element"] == 1 else _lib.DTYPE_BF16)
        need = lib.dsa_paged_attention_workspace_bytes(ctypes.addressof(cache), c["sequences"], c["tokens"], c["heads"],
                                                       c["columns"], c["uniform"])
        assert need == (COUNTERS * 4 + parts * (c["dim"] + 2) * 4 + rows * 8 if parts else 0), c
        group = c["heads"] // c["kv_heads"]
        done: dict[int, int] = {}
        for launch in launches:
            pieces = _pieces(launch, group, c["spans"], c["keys"])
            assert len(pieces) <= launch["grid"], (c, launch)
            seen: dict[tuple, list] = {}
            slots = set()
            for b, tile, first, long, slot, count in pieces:
                seen.setdefault((b, tile), []).append((first, long, count))
                done[b] = max(done.get(b, 0), min(c["spans"][b] * group, (tile + 1) * launch["tile"]))
                if count > 1:
                    at = slot + first // long
                    assert at not in slots and (at + 1) * c["kv_heads"] * launch["rows"] <= parts, (c, launch)
                    slots.add(at)
                    assert launch["cuts"] and count <= MOST_SPLITS
                    if launch["counts"]:
                        assert (slot + 1) * launch["kinds"] <= COUNTERS, (c, launch)
            for (b, _), found in seen.items():
                units = _up(c["keys"][b], launch["unit"])
                assert len(found) == found[0][2]
                covered = [u for first, long, _ in found for u in range(first, min(first + long, units))]
                assert covered == list(range(units)), (c, launch)
        for b, n in enumerate(c["spans"]):  # by exactly one launch, which takes all of its rows
            takers = [x for x in launches if x["least"] <= n * group <= x["most"]]
            assert len(takers) == (1 if n else 0) and done.get(b, 0) == n * group, c
