"""Cache rows of positions through a page table: real ones and padding."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from dsa_amd import paged

TABLE = torch.tensor([[3, 1, 0], [7, 2, 0]], dtype=torch.int32)  # unused columns are zeros


@pytest.mark.parametrize("size", [1, 4, 64])
def test_rows_of_positions(size) -> None:
    cache = SimpleNamespace(page_size=size)
    positions = torch.arange(3 * size).repeat(2)
    sequences = torch.tensor([0, 1]).repeat_interleave(3 * size)
    want = [int(TABLE[s, p // size]) * size + p % size for s, p in zip(sequences.tolist(), positions.tolist())]
    for dtype in (torch.int64, torch.int32):
        got = paged.cache_rows(cache, TABLE, positions.to(dtype), sequences.to(dtype))
        assert got.dtype == torch.int64 and got.tolist() == want
    assert paged.cache_rows(cache, TABLE, torch.tensor([size, 0])).tolist() == [size, 7 * size]


@pytest.mark.parametrize("size", [1, 4, 64])
def test_padding_has_no_row(size) -> None:
    """Neither a position of -1 nor one past the table wraps into a page of it."""

    cache = SimpleNamespace(page_size=size)
    assert paged.cache_rows(cache, TABLE, torch.tensor([-1, size - 1])).tolist() == [-1, 8 * size - 1]
    positions = torch.tensor([0, -1, -size - 5, 3 * size, 2**40, -(2**62), 0, 0, 0])
    sequences = torch.tensor([1, 1, 0, 0, 0, 1, -1, 2, 2**40])
    assert paged.cache_rows(cache, TABLE, positions, sequences).tolist() == [7 * size] + [-1] * 8
    assert paged.cache_rows(cache, TABLE[:, :0], torch.tensor([0, -1])).tolist() == [-1, -1]


def test_refusals() -> None:
    cache = SimpleNamespace(page_size=16)
    with pytest.raises(ValueError, match="one token per sequence"):
        paged.cache_rows(cache, TABLE, torch.tensor([0]))
    with pytest.raises(ValueError, match="page_table"):
        paged.cache_rows(cache, TABLE[0], torch.tensor([0]))


@pytest.mark.gpu
def test_padding_is_not_appended(device) -> None:
    """Tokens of position -1 leave every row of the cache as it was."""

    cache = paged.new_cache(8, 16, 2, 64, device=device)
    cache.keys.fill_(5.0)
    cache.values.fill_(6.0)
    table = TABLE.to(device)
    positions = torch.tensor([17, -1, -1, 3], device=device)
    sequences = torch.tensor([0, 0, 1, 1], device=device)
    rows = paged.cache_rows(cache, table, positions, sequences)
    new = torch.randn(4, 2, 64, dtype=torch.bfloat16, device=device)
    paged.append(cache, new, new, rows, positions, rope_dim=0)
    keys, values = cache.keys.view(-1, 2, 64), cache.values.view(-1, 2, 64)
    written = [1 * 16 + 1, 7 * 16 + 3]
    assert torch.equal(keys[written], new[[0, 3]]) and torch.equal(values[written], new[[0, 3]])
    others = [r for r in range(8 * 16) if r not in written]
    assert (keys[others] == 5.0).all() and (values[others] == 6.0).all()
