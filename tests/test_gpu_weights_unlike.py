"""Accumulated weights of batches whose sequences are of very unlike lengths, at sizes
where the long one is dealt to several workgroups, each with many steps.  Bounds as in
``test_gpu_eviction``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dsa_amd import eviction, paged
from oracle import eviction as oracle
from test_gpu_eviction import _case
from test_gpu_paged import BF16, F16, FP8, _f64
from test_gpu_paged_fp4 import FP4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,chunks,group,kv_heads,dim,dtype,starts", [
    ([64] * 255 + [40000], [1] * 256, 4, 2, 64, BF16, False),
    ([64] * 100 + [40000] + [63] * 155, [1] * 256, 2, 2, 64, FP4, True),    # most rows are single tokens'
    ([40000] + [1, 0, 200] * 40, [100] + [1, 0, 3] * 40, 4, 1, 64, F16, True),  # the long one is a chunk
    ([30001] + [9] * 63, [40] + [1] * 63, 2, 1, 128, FP8, True),
    ([50000, 33], [1, 1], 8, 1, 128, FP4, False),
    ([20000] + [17] * 30, [2] * 31, 1, 8, 256, BF16, False),
])
def test_one_long_sequence_among_short_ones(device, lengths, chunks, group, kv_heads, dim, dtype, starts) -> None:
    print(f"weights of unlike lengths: {len(lengths)} to {max(lengths)} x {group}/{kv_heads}x{dim} {dtype}", flush=True)
    c = _case(device, 110, lengths, chunks, group * kv_heads, kv_heads, dim, 16, dtype)
    q, args = c.q.to(device), c.device_args(starts=starts)
    _, lse = paged.attention(q, c.cache, *args, return_lse=True)
    weights = eviction.new_weights(c.cache)
    eviction.accumulate_weights(weights, q, c.cache, *args[:2], lse, args[2])
    want, off = oracle.added_weights(_f64(c.q), np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts,
                                     lse.double().cpu().numpy(), dim**-0.5)
    assert (np.abs(weights.double().cpu().numpy() - want) <= off).all()
    again = eviction.new_weights(c.cache)
    eviction.accumulate_weights(again, q, c.cache, *args[:2], lse, args[2])
    assert torch.equal(again, weights)
