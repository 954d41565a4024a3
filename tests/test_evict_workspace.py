"""The eviction's workspace follows what the work can reach."""

from __future__ import annotations

import ctypes

import pytest

from dsa_amd import _lib
from test_paged_api import _descriptor


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
