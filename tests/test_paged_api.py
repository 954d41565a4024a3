"""The paged cache's entry points without a device: refusals of the C entries,
the descriptor's layout and the oracle's own identities."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from dsa_amd import _lib, paged
from oracle import paged as oracle


def _descriptor(**kw) -> _lib.PagedCacheC:
    fields = dict(keys=256, values=256, key_scales=256, value_scales=256, pages=8, key_page_stride=4096,
                  key_slot_stride=256, key_head_stride=128, value_page_stride=4096, value_slot_stride=256,
                  value_head_stride=128, page_size=16, kv_heads=2, head_dim=128, dtype=_lib.DTYPE_BF16)
    fields.update(kw)
    return _lib.PagedCacheC(**fields)


def test_descriptor_matches_the_header() -> None:
    assert ctypes.sizeof(_lib.PagedCacheC) == 4 * 8 + 7 * 8 + 4 * 4
    assert _lib.PagedCacheC.pages.offset == 32 and _lib.PagedCacheC.page_size.offset == 88


@pytest.mark.parametrize("fields,message", [
    ({"keys": None}, b"no keys"),
    ({"dtype": _lib.DTYPE_F32}, b"bf16, fp16 or fp8"),
    ({"dtype": _lib.DTYPE_FP8_E4M3, "key_scales": None}, b"scales"),
    ({"page_size": 24}, b"page_size"),
    ({"page_size": 0}, b"page_size"),
    ({"head_dim": 96}, b"head_dim"),
    ({"kv_heads": 0}, b"kv_heads"),
    ({"pages": 0}, b"pages"),
    ({"pages": 1 << 28}, b"pages"),
    ({"key_slot_stride": 129}, b"16 bytes"),
    ({"value_page_stride": -8}, b"non-negative"),
    ({"key_page_stride": 1 << 33}, b"4 GiB"),
    ({"values": 264}, b"aligned"),
])
def test_descriptors_are_refused(fields, message) -> None:
    lib = _lib.load()
    d = _descriptor(**fields)
    fake = ctypes.c_void_p(256)
    at = ctypes.addressof(d)
    assert lib.dsa_paged_append(at, fake, 256, fake, 256, None, 0, None, 0, 2, fake, fake, 1, 128, 10000.0, None) == 1
    assert message in lib.dsa_last_error()
    assert lib.dsa_paged_attention(at, fake, 512, fake, 4, 4, fake, None, 1, 1, 4, 2, 1.0, 1, fake, None, None, 0, None) == 1
    assert message in lib.dsa_last_error()


def _append(lib, d, **kw):
    a = dict(keys=256, ks=256, values=256, vs=256, q=None, qs=0, out=None, heads=0, dtype=2, rows=256, positions=256,
             tokens=1, rope=128, theta=10000.0)
    a.update(kw)
    return lib.dsa_paged_append(ctypes.addressof(d), a["keys"], a["ks"], a["values"], a["vs"], a["q"], a["qs"], a["out"],
                                a["heads"], a["dtype"], a["rows"], a["positions"], a["tokens"], a["rope"], a["theta"], None)


@pytest.mark.parametrize("args,message", [
    ({"keys": None}, b"null"), ({"rows": None}, b"null"), ({"tokens": -1}, b"tokens"), ({"dtype": 0}, b"bf16 or fp16"),
    ({"dtype": 1}, b"cache's type"), ({"rope": 136}, b"rope_dim"), ({"rope": 24}, b"rope_dim"), ({"theta": 0.0}, b"theta"),
    ({"theta": float("inf")}, b"theta"), ({"ks": 255}, b"strides"), ({"vs": 128}, b"strides"), ({"values": 264}, b"aligned"),
    ({"q": 256}, b"output"), ({"q": 256, "out": 256, "heads": 4, "qs": 8}, b"strides"),
])
def test_append_refuses(args, message) -> None:
    lib = _lib.load()
    assert _append(lib, _descriptor(), **args) == 1
    assert message in lib.dsa_last_error()


def test_append_of_no_tokens_is_accepted() -> None:
    assert _append(_lib.load(), _descriptor(), tokens=0, keys=None) == 0


def _attend(lib, d, selected, **kw):
    a = dict(q=256, qs=512, table=256, ts=4, cols=4, lengths=256, starts=None, seqs=1, tokens=1, heads=4, dtype=2, out=256,
             ws=None, bytes=0, idx=256, istride=64, k=64)
    a.update(kw)
    head = (ctypes.addressof(d), a["q"], a["qs"], a["table"], a["ts"], a["cols"], a["lengths"], a["starts"], a["seqs"],
            a["tokens"], a["heads"], a["dtype"])
    if selected:
        return lib.dsa_paged_selected_attention(*head, a["idx"], a["istride"], a["k"], 1.0, a["out"], None, a["ws"],
                                                a["bytes"], None)
    return lib.dsa_paged_attention(*head, 1.0, 1, a["out"], None, a["ws"], a["bytes"], None)


@pytest.mark.parametrize("selected", [False, True])
@pytest.mark.parametrize("args,message", [
    ({"q": None}, b"null"), ({"table": None}, b"null"), ({"lengths": None}, b"null"), ({"out": None}, b"null"),
    ({"seqs": 0}, b"sequences"), ({"tokens": -1}, b"tokens"), ({"heads": 3}, b"evenly"), ({"heads": 0}, b"evenly"),
    ({"dtype": 0}, b"bf16 or fp16"), ({"dtype": 1}, b"cache's type"), ({"seqs": 2}, b"as many tokens"),
    ({"cols": 0}, b"columns"), ({"ts": 3}, b"columns"), ({"qs": 500}, b"query_stride"), ({"q": 264}, b"aligned"),
])
def test_attention_refuses(selected, args, message) -> None:
    lib = _lib.load()
    assert _attend(lib, _descriptor(), selected, **args) == 1
    assert message in lib.dsa_last_error()


def test_selected_refuses_bad_lists_and_small_workspaces() -> None:
    lib = _lib.load()
    d = _descriptor()
    for bad in ({"idx": None}, {"istride": 63}, {"k": -1}):
        assert _attend(lib, d, True, **bad) == 1
        assert b"index lists" in lib.dsa_last_error()
    at = ctypes.addressof(d)
    need = lib.dsa_paged_selected_workspace_bytes(at, 1, 4, 2048)
    assert need > 0
    assert _attend(lib, d, True, k=2048, istride=2048, ws=256, bytes=need - 1) == 3
    need = lib.dsa_paged_attention_workspace_bytes(at, 1, 1, 4, 128, 1)
    assert need > 0 and lib.dsa_paged_attention_workspace_bytes(at, 1, 0, 4, 128, 1) == 0
    assert _attend(lib, d, False, cols=128, ts=128, ws=256, bytes=need - 1) == 3
    assert _attend(lib, d, False, cols=128, ts=128, ws=264, bytes=need) == 3


def test_host_tensors_are_refused() -> None:
    x = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensors"):
        paged.PagedCache(x, x)


def test_oracle_attention_is_a_softmax_average() -> None:
    rng = np.random.default_rng(0)
    keys, values = rng.normal(size=(3, 4, 2, 8)), rng.normal(size=(3, 4, 2, 8))
    q = rng.normal(size=(2, 4, 8))
    table = np.array([[2, 0, 1]])
    out, lse, _, _ = oracle.attention(q, keys, values, table, [10], [0, 2], 0.5)
    k, v = keys[[2, 0, 1]].reshape(12, 2, 8)[:9], values[[2, 0, 1]].reshape(12, 2, 8)[:9]
    w = np.exp(0.5 * k[:, 1] @ q[0, 3])
    assert np.allclose(out[0, 3], w @ v[:, 1] / w.sum()) and np.isclose(lse[0, 3], np.log(w.sum()))
    lists = np.tile(np.arange(9), (2, 1))
    same = oracle.attention(q, keys, values, table, [10], [0, 2], 0.5, lists=lists)
    assert np.allclose(same[0][0], out[0])


def test_oracle_rotation_keeps_lengths_and_relative_angles() -> None:
    rng = np.random.default_rng(1)
    x, y = rng.normal(size=(1, 1, 16)), rng.normal(size=(1, 1, 16))
    at = lambda v, p: oracle.rotate(v, np.array([p]), 8, 100.0)[0, 0]  # noqa: E731
    assert np.isclose(np.linalg.norm(at(x, 77)), np.linalg.norm(x))
    assert np.isclose(at(x, 105) @ at(y, 100), at(x, 1005) @ at(y, 1000))
    assert np.array_equal(at(x, 5)[8:], x[0, 0, 8:])


def test_command_line_of_attend(tmp_path) -> None:
    from dsa_amd.cli import build_parser

    parser = build_parser()
    args = parser.parse_args(["attend", "--output", str(tmp_path), "--cache-dtype", "fp8", "--k", "64"])
    assert (args.length, args.steps, args.k, args.head_dim, args.cache_dtype) == (16384, 16, 64, 128, "fp8")
    for bad in (["--cache-dtype", "int4"], ["--head-dim", "96"]):
        with pytest.raises(SystemExit):
            parser.parse_args(["attend", "--output", str(tmp_path), *bad])
    with pytest.raises(ValueError, match="at least 1"):
        args.steps = 0
        args.function(args)
