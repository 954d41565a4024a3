"""A 4-bit cache of a caller's own may have any power of two that a byte holds: what rows
under the least and the largest ones stand for, and that values past bf16 (infinite
there) reach the rows that see them and no others."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from dsa_amd import paged
from oracle import paged as oracle
from test_gpu_paged import BF16, _f64
from test_gpu_paged_fp4 import E8M0, FP4, Case4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_read_of_every_code_under_every_power(device, dim) -> None:
    """Exact in bf16, subnormal ones too; values from 2^128 on are infinite."""

    print(f"every power, {dim} dims", flush=True)
    pages, page, kv_heads = 8, 32, 2
    powers = torch.arange(256, dtype=torch.uint8).view(pages, page)[:, None, :, None].expand(-1, kv_heads, -1, dim // 32)
    codes = torch.arange(dim // 2, dtype=torch.uint8) * 37  # every pair of codes within 256 bytes
    codes = codes + torch.arange(kv_heads, dtype=torch.uint8)[:, None] * 128
    codes = codes.expand(pages, page, -1, -1).contiguous()
    want = torch.from_numpy(oracle.fp4_values(codes.numpy(), powers.transpose(1, 2).numpy())).flatten(0, 1)
    cache = paged.PagedCache(*(codes.to(device).view(FP4) for _ in range(2)),
                             *(powers.contiguous().to(device).view(E8M0) for _ in range(2)))
    for got in paged.read(cache, torch.arange(256, device=device)):
        got = got.double().cpu()
        assert torch.isnan(got[255]).all() and torch.isnan(want[255]).all()
        far = want[:255].abs() >= 2.0**128
        assert torch.isinf(got[:255][far]).all() and torch.equal(got[:255][far].sign(), want[:255][far].sign())
        assert far.any() and torch.equal(got[:255][~far], want[:255][~far])


@pytest.mark.parametrize("power,code", [(252, 7), (253, 6), (253, 14), (253, 7), (254, 4), (254, 15), (255, 0)])
@pytest.mark.parametrize("lengths,chunks,heads,kv_heads,dim", [
    ([90], [3], 4, 2, 128), ([200, 40], [30, 30], 8, 2, 64), ([333], [200], 8, 2, 128), ([150], [40], 4, 1, 256),
    ([2500], [2], 4, 4, 64), ([300], [90], 16, 1, 128), ([300], [300], 8, 1, 64),
])
def test_values_past_bf16_reach_the_rows_that_see_them_alone(device, lengths, chunks, heads, kv_heads, dim, power, code) -> None:
    """A block of a later token's value, every second dim 0: infinite (or, past fp32's
    range under a softmax's weights, overflowing) dims in the rows that see it, and bits
    as without it everywhere else."""

    print(f"power {power} code {code}: {lengths} {chunks} {heads}/{kv_heads}x{dim}", flush=True)
    c = Case4(device, 31, lengths, chunks, heads, kv_heads, dim, 16)
    n, new = lengths[0], chunks[0]
    at = n - new + new // 2  # seen by the last new tokens of the first sequence
    row = int(paged.cache_rows(c.cache, c.table.to(device), torch.tensor([at], device=device),
                               torch.zeros(1, dtype=torch.int64, device=device)))
    block = c.cache.values.view(torch.uint8)[row // 16, row % 16, kv_heads - 1, 16:32]
    block.zero_()
    want, want_lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
    block.fill_(code << 4)
    c.cache.value_scales.view(torch.uint8)[row // 16, kv_heads - 1, row % 16, 1] = power
    got, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
    hit = torch.zeros(got.shape, dtype=torch.bool, device=device)
    hit[new // 2:new, (kv_heads - 1) * (heads // kv_heads):, 32:64] = True
    if power < 255:
        hit[..., ::2] = False
        if power > 252:
            assert torch.isinf(got[hit]).all() and ((got[hit] < 0) == (code > 7)).all()
    else:
        assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], want[~hit])
    assert torch.equal(lse, want_lse)


@pytest.mark.parametrize("power", [0, 1, 200])
def test_attention_to_values_far_from_1(device, power) -> None:
    """Subnormal ones, and the largest whose sums under a softmax's weights (2^14 at
    most) stay in fp32's range."""

    c = Case4(device, 40, [70], [9], 4, 2, 64, 16)
    store = c.cache.value_scales.view(torch.uint8)
    spread = torch.randint(0, 3, store.shape, generator=c.gen, dtype=torch.uint8)
    store.copy_(spread.to(device) + power)
    c.values64 = oracle.fp4_values(c.cache.values.view(torch.uint8).cpu().numpy(), store.transpose(1, 2).cpu().numpy())
    out, lse = paged.attention(c.q.to(device), c.cache, *c.device_args(), return_lse=True)
    ref, _, weighted, sizes = oracle.attention(_f64(c.q), c.keys64, c.values64, c.table.numpy(), c.lengths, c.starts, 64**-0.5)
    # the weights' and the output's rounding to bf16, of which the last has steps of 2^-133 at least
    assert (np.abs(_f64(out) - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-7 * weighted + 2.0**-133).all()
    assert out.dtype == BF16
