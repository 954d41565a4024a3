"""Accumulated weights where scores are infinite: a row whose every score is -inf has no
softmax weight to give, as it has no output, and leaves the other rows' sums alone."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsa_amd import eviction, paged
from oracle import eviction as oracle
from test_gpu_eviction import _case
from test_gpu_paged import BF16, F16, FP8, _f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,dtype", [
    ([70], [1], 8, 2, 128, BF16),             # few rows
    ([90, 33], [3, 2], 8, 2, 64, F16),
    ([300], [300], 8, 2, 128, BF16),          # many, and pieces of them
    ([700, 300], [200, 200], 6, 2, 64, F16),
    ([400, 50, 9], [150, 1, 1], 4, 1, 256, BF16),  # a chunk among single tokens
])
def test_rows_whose_scores_are_all_minus_infinity(device, lengths, chunks, heads, kv_heads, dim, dtype, causal) -> None:
    """Dim 0 of every key is 1/2; a dead row's is -inf, and 0 its others."""

    print(f"-inf: {lengths} {chunks} {heads}/{kv_heads}x{dim} {dtype} {causal}", flush=True)
    c = _case(device, 21, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    gen = torch.Generator().manual_seed(3)
    args = c.device_args()
    dead = torch.rand(c.q.shape[:2], generator=gen) < 0.3
    dead[0, 0] = True
    c.q[dead] = 0
    c.q[..., 0] = torch.where(dead, -math.inf, 1.0)
    c.cache.keys[..., 0] = 0.5
    q, on_device = c.q.to(device), dead.to(device)
    out, lse = paged.attention(q, c.cache, *args, causal=causal, return_lse=True)
    assert (out[on_device] == 0).all() and (lse[on_device] == -math.inf).all()
    got = eviction.new_weights(c.cache)
    eviction.accumulate_weights(got, q, c.cache, *args[:2], lse, args[2], causal=causal)
    keys = np.nan_to_num(c.keys64)
    keys[..., 0] = 0.5
    sums = lse.double().cpu().numpy()
    sums[dead.numpy()] = 1e4  # exp(0 - 1e4) = 0
    alive = _f64(c.q)
    alive[dead.numpy()] = 0
    want, off = oracle.added_weights(alive, keys, c.table.numpy(), lengths, c.starts, sums, dim**-0.5, causal=causal)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all() and (np.abs(got - want) <= off).all()


@pytest.mark.parametrize("chunk", [2, 90])
def test_rows_of_fp8_keys(device, chunk) -> None:
    """e4m3 keys, whose scales come after the product."""

    c = _case(device, 22, [200], [chunk], 4, 2, 128, 16, FP8)
    q, args = c.q.to(device), c.device_args()
    q[0] = 0
    q[0, :, 0] = -math.inf
    c.cache.keys.view(torch.uint8)[..., 0] = 0x38  # 1
    out, lse = paged.attention(q, c.cache, *args, return_lse=True)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    got, want = eviction.new_weights(c.cache), eviction.new_weights(c.cache)
    eviction.accumulate_weights(got, q, c.cache, *args[:2], lse, args[2])
    eviction.accumulate_weights(want, q[1:], c.cache, *args[:2], lse[1:], args[2] - torch.tensor([0, 1], device=device, dtype=torch.int32))
    assert torch.isfinite(got).all() and torch.allclose(got, want, rtol=2.0**-18, atol=0)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim,dtype", [
    ([70], [1], 8, 2, 128, BF16), ([300], [300], 8, 2, 128, BF16), ([2000], [700], 4, 1, 64, F16),
    ([400, 50, 9], [150, 1, 1], 4, 1, 256, BF16), ([900], [300], 8, 2, 128, FP8), ([90, 33], [3, 2], 8, 2, 64, FP8),
])
def test_rows_without_a_log_sum_add_nothing_whatever_they_hold(device, lengths, chunks, heads, kv_heads, dim, dtype, causal) -> None:
    """A log sum of -inf leaves a row out: its query may be NaN."""

    print(f"left out: {lengths} {chunks} {heads}/{kv_heads}x{dim} {dtype} {causal}", flush=True)
    c = _case(device, 23, lengths, chunks, heads, kv_heads, dim, 16, dtype)
    args = c.device_args()
    _, lse = paged.attention(c.q.to(device), c.cache, *args, causal=causal, return_lse=True)
    out = torch.rand(c.q.shape[:2], generator=torch.Generator().manual_seed(4)) < 0.02
    out[0, 0] = out[-1, -1] = True
    q = c.q.clone()
    q[out] = math.nan
    lse = lse.masked_fill(out.to(device), -math.inf)
    got = eviction.new_weights(c.cache)
    eviction.accumulate_weights(got, q.to(device), c.cache, *args[:2], lse, args[2], causal=causal)
    sums, kept = lse.double().cpu().numpy(), _f64(c.q)
    sums[out.numpy()], kept[out.numpy()] = 1e4, 0
    want, off = oracle.added_weights(kept, np.nan_to_num(c.keys64), c.table.numpy(), lengths, c.starts, sums, dim**-0.5,
                                     causal=causal)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all() and (np.abs(got - want) <= off).all()
