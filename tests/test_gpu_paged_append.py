"""The rotation of appended keys far into a context: the scales and values of an fp8
cache against float64, where an angle taken as an fp32 product is off by up to
0.0006 rad."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dsa_amd import paged
from oracle import paged as oracle
from test_gpu_paged import BF16, F16, FP8, _f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,rope_dim", [(FP8, 128, 64), (FP8, 64, 64), (BF16, 128, 128), (F16, 256, 128)])
@pytest.mark.parametrize("start", [0, 9000, 33000, 65535, 1 << 20])
def test_positions_far_into_a_context(device, start, dtype, dim, rope_dim) -> None:
    tokens, kv_heads, page = 601, 4, 32
    gen = torch.Generator().manual_seed(start + dim)
    cache = paged.new_cache(20, page, kv_heads, dim, dtype=dtype, device=device)
    keys, values = (torch.randn(tokens, kv_heads, dim, generator=gen).to(cache.row_dtype) for _ in range(2))
    positions = torch.arange(start, start + tokens)
    rows = torch.randperm(cache.rows, generator=gen)[:tokens]
    paged.append(cache, keys.to(device), values.to(device), rows.to(device), positions.to(device), rope_dim=rope_dim)
    turned = oracle.rotate(_f64(keys), positions.numpy(), rope_dim, 10_000.0)
    got = _f64(cache.keys).reshape(-1, kv_heads, dim)[rows.numpy()]
    # fp32: the angle, reduced in double, to 2^-23, its sine and cosine, two products and a sum
    slack = 2.0**-21 * np.abs(_f64(keys)).max(axis=-1, keepdims=True)
    if dtype == FP8:
        scales = cache.key_scales.cpu().double().numpy().reshape(-1, kv_heads)[rows.numpy()]
        want = oracle.head_scale(turned)
        assert np.linalg.norm(scales - want) <= 1e-6 * np.linalg.norm(want)
        bound = 2.0**-4 * np.abs(turned) + 2.0**-10 * scales[..., None] + slack  # half of an e4m3 step
        assert (np.abs(got * scales[..., None] - turned) <= bound).all()
    else:
        unit = 2.0**-8 if dtype == BF16 else 2.0**-11
        assert (np.abs(got - turned) <= unit * np.abs(turned) + slack).all()
