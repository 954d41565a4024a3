"""The 4-bit cache's entry points without a device: refusals of the C entries and the
oracle's own identities."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from dsa_amd import _lib
from oracle import paged as oracle
from test_eviction_api import _weights
from test_paged_api import _append, _attend, _descriptor

FP4 = _lib.DTYPE_FP4_E2M1


def _read(lib, d, **kw):
    a = dict(rows=256, count=1, keys=256, values=256)
    a.update(kw)
    return lib.dsa_paged_read(ctypes.addressof(d), a["rows"], a["count"], a["keys"], a["values"], None)


@pytest.mark.parametrize("args,message", [
    ({"rows": None}, b"null"), ({"count": -1}, b"rows"), ({"count": 1 << 31}, b"rows"), ({"keys": 264}, b"aligned"),
    ({"values": 264}, b"aligned"), ({"count": (1 << 31) - 1}, b"too many rows"),
])
def test_read_refuses(args, message) -> None:
    lib = _lib.load()
    assert _read(lib, _descriptor(), **args) == 1
    assert message in lib.dsa_last_error()


def test_read_of_nothing_is_accepted() -> None:
    lib = _lib.load()
    assert _read(lib, _descriptor(), count=0, rows=None) == 0
    assert _read(lib, _descriptor(), keys=None, values=None) == 0


@pytest.mark.parametrize("fields,message", [
    ({"key_scales": None}, b"scales"), ({"value_scales": None}, b"scales"), ({"key_scales": 264}, b"aligned"),
    ({"value_scales": 264}, b"aligned"),
])
def test_descriptors_of_4_bits_are_refused(fields, message) -> None:
    lib = _lib.load()
    d = _descriptor(**{"dtype": FP4, "key_scales": 256, "value_scales": 256, **fields})
    for call in (_append, _read, _weights, lambda *a: _attend(*a, False), lambda *a: _attend(*a, True)):
        assert call(lib, d) == 1
        assert message in lib.dsa_last_error()


def test_4_bits_take_bf16_alone() -> None:
    lib = _lib.load()
    d = _descriptor(dtype=FP4, key_scales=256, value_scales=256)
    for call in (_append, _weights):
        assert call(lib, d, dtype=1) == 1
        assert b"bf16" in lib.dsa_last_error()
    for selected in (False, True):
        assert _attend(lib, d, selected, dtype=1) == 1
        assert b"bf16" in lib.dsa_last_error()


def test_weights_of_too_many_rows_are_refused() -> None:
    lib = _lib.load()
    assert _weights(lib, _descriptor(), tokens=(1 << 28) - 1, heads=64, qs=8192) == 1
    assert b"too many" in lib.dsa_last_error()


def test_oracle_blocks_are_within_half_a_step() -> None:
    x = np.random.default_rng(0).normal(size=(64, 2, 64)) * 2.0 ** np.arange(-32, 32)[:, None, None]
    y, powers = oracle.fp4(x)
    blocks = np.abs(x).reshape(64, 2, 2, 32).max(-1)
    step = 2.0 ** (powers.astype(np.int64).reshape(64, 2, 2) - 127)
    assert (blocks <= 7 * step).all() and (blocks > 3.5 * step).all()
    off = np.abs(x - y).reshape(64, 2, 2, 32) / step[..., None]
    size = np.abs(x).reshape(64, 2, 2, 32) / step[..., None]
    assert (off <= np.where(size < 2, 0.25, np.where(size < 4, 0.5, 1.0))).all()
