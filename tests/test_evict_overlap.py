"""``dsa_paged_evict`` refuses new lengths that lie over the old ones, which its later
workgroups still read; lengths side by side are taken."""

from __future__ import annotations

import pytest
import torch

from dsa_amd import _lib, eviction, paged
from test_eviction_api import _evict
from test_paged_api import _descriptor


@pytest.mark.parametrize("per_head", [0, 1])
@pytest.mark.parametrize("lengths,out,seqs", [(256, 256, 1), (256, 256, 5), (256, 260, 2), (260, 256, 2), (256, 272, 5)])
def test_overlapping_lengths_are_refused(lengths, out, seqs, per_head) -> None:
    lib = _lib.load()
    assert _evict(lib, _descriptor(), lengths=lengths, out=out, seqs=seqs, per_head=per_head) == 1
    assert b"out_lengths must not overlap" in lib.dsa_last_error()


@pytest.mark.gpu
def test_lengths_side_by_side(device) -> None:
    cache = paged.new_cache(4, 16, 2, 64, device=device)
    cache.keys.zero_(), cache.values.zero_()
    weights = eviction.new_weights(cache)
    table = torch.arange(4, dtype=torch.int32, device=device).view(2, 2)
    both = torch.tensor([30, 20, -1, -1], dtype=torch.int32, device=device)
    kept = torch.empty(2, 2, 24, dtype=torch.int64, device=device)
    need = _lib.query("dsa_paged_evict_workspace_bytes", cache._address, 2, 2, 24, 1)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call("dsa_paged_evict", cache._address, table.data_ptr(), 2, 2, both.data_ptr(), 2, weights.data_ptr(), 24, 0, 1,
              both[2:].data_ptr(), kept.data_ptr(), workspace.data_ptr(), need, _lib.stream_of(weights))
    assert both.tolist() == [30, 20, 24, 20]
