"""The eviction's workspace follows what the work can reach: the moves that a list can
make, and the lists that the cache's rows can make long."""

from __future__ import annotations

import ctypes

import pytest
import torch

from dsa_amd import _lib, eviction, paged
from test_paged_api import _descriptor

LONG = 16384  # positions of a list that one workgroup holds
CHUNK = 8192  # and of a longer one's chunks


def _need(d, sequences, columns, keep, per_head) -> int:
    return _lib.query("dsa_paged_evict_workspace_bytes", ctypes.addressof(d), sequences, columns, keep, per_head)


@pytest.mark.parametrize("per_head", [0, 1])
@pytest.mark.parametrize("sequences,columns,keep", [
    (1, 260, 4096), (256, 260, 4096), (256, 260, 64), (3, 4, 63), (3, 4, 64), (3, 4, 65), (7, 1024, 1), (2, 4, 1 << 30),
])
def test_moves_that_a_list_can_make(sequences, columns, keep, per_head) -> None:
    """As many as it keeps, or as lie past those: 64 of 4160 keys that are cut to 4096,
    none where nothing can be evicted."""

    d = _descriptor(pages=512)  # 8192 rows: no list is long
    lists = sequences * (2 if per_head else 1)
    moves = max(0, min(keep, 16 * columns - keep))
    need = _need(d, sequences, columns, keep, per_head)
    assert 0 < need <= lists * (8 * moves + 64) + 64

@pytest.mark.parametrize("per_head", [0, 1])
@pytest.mark.parametrize("pages,sequences,columns", [(1 << 16, 256, 8192), (1 << 16, 1, 8192), (2000, 20000, 2000), (1 << 20, 4, 65536)])
def test_lists_that_can_be_long(pages, sequences, columns, per_head) -> None:
    d = _descriptor(pages=pages)
    heads = 2 if per_head else 1
    lists, rows, keep = sequences * heads, 16 * pages, 16
    chunks = heads * min(sequences * -(-16 * columns // CHUNK), 3 * rows // LONG)
    long = min(lists, chunks // 3)
    need = _need(d, sequences, columns, keep, per_head)
    assert 0 < need <= lists * (8 * keep + 64) + long * (3 * 2048 * 4 + 64) + chunks * (CHUNK * 4 + 16) + 256


@pytest.mark.gpu
@pytest.mark.parametrize("per_head", [0, 1])
@pytest.mark.parametrize("lengths,columns,keep", [
    ([64, 20, 0], 4, 32), ([64, 64], 4, 1), ([64, 5], 4, 63), ([64, 64], 4, 64), ([300, 65], 40, 200),
    ([16400, 40000, 300, 16385], 3000, 8000), ([33000, 16384], 2100, 32900), ([17000, 17000, 17000, 9], 1200, 3),
])
def test_nothing_is_written_past_the_workspace(device, lengths, columns, keep, per_head) -> None:
    """As many moves as there can be: weights that rise with the position keep the last."""

    print(f"workspace: {lengths} {columns} {keep} {per_head}", flush=True)
    used = [-(-n // 16) for n in lengths]
    cache = paged.new_cache(sum(used) + 1, 16, 2, 64, device=device)
    cache.keys.zero_(), cache.values.zero_()
    table = torch.zeros(len(lengths), columns, dtype=torch.int32)
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(n) + sum(used[:b])
    weights = torch.arange(cache.rows, device=device).float().expand(2, -1).contiguous()
    table, n = table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)
    out = torch.empty_like(n)
    kept = torch.empty(len(lengths), 2 if per_head else 1, keep, dtype=torch.int64, device=device)
    need = _need(cache._struct, len(lengths), columns, keep, per_head)
    workspace = torch.full((need + 65536,), 0xa5, dtype=torch.uint8, device=device)
    _lib.call("dsa_paged_evict", cache._address, table.data_ptr(), columns, columns, n.data_ptr(), len(lengths),
              weights.data_ptr(), keep, 0, per_head, out.data_ptr(), kept.data_ptr(), workspace.data_ptr(), need,
              _lib.stream_of(weights))
    assert (workspace[need:] == 0xa5).all()
    assert out.tolist() == [min(x, keep) for x in lengths]
    for b, x in enumerate(lengths):  # the last `keep`: those below m where they were, the others in order before them
        m = min(x, keep)
        first = x - m  # the first that is kept
        stay = list(range(first, m))
        want = (list(range(max(m, first), x)) + stay) if x > m else stay
        for g in range(kept.shape[1]):
            assert kept[b, g, :m].tolist() == want and (kept[b, g, m:] == -1).all()
