"""The eviction entry points without a device: refusals of the C entries and the
oracle's own identities."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from dsa_amd import _lib
from oracle import eviction as oracle
from oracle import paged as paged_oracle
from test_paged_api import _descriptor


def _weights(lib, d, **kw):
    a = dict(q=256, qs=512, table=256, ts=4, cols=4, lengths=256, starts=None, seqs=1, tokens=1, heads=4, dtype=2, lse=256,
             weights=256, ws=None, bytes=0)
    a.update(kw)
    return lib.dsa_paged_weights(ctypes.addressof(d), a["q"], a["qs"], a["table"], a["ts"], a["cols"], a["lengths"],
                                 a["starts"], a["seqs"], a["tokens"], a["heads"], a["dtype"], 1.0, 1, a["lse"],
                                 a["weights"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("args,message", [
    ({"q": None}, b"null"), ({"table": None}, b"null"), ({"lengths": None}, b"null"), ({"lse": None}, b"null"),
    ({"weights": None}, b"null"), ({"seqs": 0}, b"sequences"), ({"tokens": -1}, b"tokens"), ({"heads": 3}, b"evenly"),
    ({"dtype": 0}, b"bf16 or fp16"), ({"dtype": 1}, b"cache's type"), ({"seqs": 2}, b"as many tokens"),
    ({"cols": 0}, b"columns"), ({"ts": 3}, b"columns"), ({"qs": 500}, b"query_stride"), ({"q": 264}, b"aligned"),
])
def test_weights_refuse(args, message) -> None:
    lib = _lib.load()
    assert _weights(lib, _descriptor(), **args) == 1
    assert message in lib.dsa_last_error()


def test_weights_of_no_tokens_and_small_workspaces() -> None:
    lib = _lib.load()
    d = _descriptor()
    assert _weights(lib, d, tokens=0) == 0
    at = ctypes.addressof(d)
    assert lib.dsa_paged_weights_workspace_bytes(at, 1, 1, 4, 4, 1) == 0
    need = lib.dsa_paged_weights_workspace_bytes(at, 1, 4096, 4, 256, 1)
    assert need > 0
    for ws, size in ((None, need), (256, need - 1), (264, need)):
        assert _weights(lib, d, tokens=4096, cols=256, ts=256, ws=ws, bytes=size) == 3


def _evict(lib, d, **kw):
    a = dict(table=256, ts=4, cols=4, lengths=256, seqs=1, weights=256, keep=8, recent=0, per_head=0, out=256, kept=256,
             ws=256, bytes=1 << 20)
    a.update(kw)
    return lib.dsa_paged_evict(ctypes.addressof(d), a["table"], a["ts"], a["cols"], a["lengths"], a["seqs"], a["weights"],
                               a["keep"], a["recent"], a["per_head"], a["out"], a["kept"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("args,message", [
    ({"table": None}, b"null"), ({"lengths": None}, b"null"), ({"weights": None}, b"null"), ({"out": None}, b"null"),
    ({"kept": None}, b"null"), ({"seqs": 0}, b"sequences"), ({"cols": 0}, b"columns"), ({"ts": 3}, b"columns"),
    ({"keep": 0}, b"keep"), ({"keep": 1 << 31}, b"keep"), ({"recent": -1}, b"recent"), ({"recent": 9}, b"recent"),
    ({"seqs": 1 << 17, "bytes": 1 << 40}, b"too many sequences"),
])
def test_evict_refuses(args, message) -> None:
    lib = _lib.load()
    assert _evict(lib, _descriptor(), **args) == 1
    assert message in lib.dsa_last_error()


def test_evict_refuses_small_workspaces_and_descriptors() -> None:
    lib = _lib.load()
    d = _descriptor()
    at = ctypes.addressof(d)
    for per_head in (0, 1):
        need = lib.dsa_paged_evict_workspace_bytes(at, 3, 4, 8, per_head)
        assert need > 0
        for ws, size in ((None, need), (256, need - 1), (264, need)):
            assert _evict(lib, d, seqs=3, per_head=per_head, ws=ws, bytes=size) == 3
    assert lib.dsa_paged_evict_workspace_bytes(at, 0, 4, 8, 0) == 0
    assert _evict(lib, _descriptor(page_size=24)) == 1
    assert _evict(lib, _descriptor(dtype=_lib.DTYPE_FP4_E2M1, value_scales=None)) == 1
    assert b"scales" in lib.dsa_last_error()


def test_oracle_weights_of_all_keys_add_up_to_the_rows() -> None:
    rng = np.random.default_rng(0)
    keys = rng.normal(size=(3, 4, 2, 8))
    q = rng.normal(size=(5, 4, 8))
    table, starts = np.array([[2, 0, 1]]), [0, 5]
    _, lse, _, _ = paged_oracle.attention(q, keys, keys, table, [10], starts, 0.5)
    w, _ = oracle.added_weights(q, keys, table, [10], starts, lse, 0.5)
    assert np.allclose(w.sum(1), 5 * 2)  # 5 tokens, 2 heads each
    assert (w.reshape(2, 3, 4)[:, 1, 2:] == 0).all()  # positions 10 and 11


def test_oracle_eviction_keeps_what_it_says() -> None:
    w = np.array([5.0, 1.0, 3.0, 3.0, np.nan, 0.0, 9.0, 0.0], dtype=np.float32)
    assert oracle.choose(w, 8, 4, 1) == [0, 6, 2, 7]
    assert oracle.choose(w, 8, 4, 0) == [0, 6, 2, 3]
    assert oracle.choose(w, 8, 3, 3) == [5, 6, 7]
    assert oracle.choose(w, 8, 7, 0) == [0, 1, 2, 3, 7, 5, 6]
    assert oracle.choose(w, 5, 8, 2) == [0, 1, 2, 3, 4]


def test_command_line_of_the_budget(tmp_path) -> None:
    from dsa_amd.cli import build_parser

    args = build_parser().parse_args(["attend", "--output", str(tmp_path), "--cache-dtype", "fp4", "--budget", "4096"])
    assert (args.cache_dtype, args.budget) == ("fp4", 4096)
    assert build_parser().parse_args(["attend", "--output", str(tmp_path)]).budget is None
    args.budget = 1
    with pytest.raises(ValueError, match="budget"):
        args.function(args)
