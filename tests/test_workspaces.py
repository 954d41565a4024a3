"""The workspaces that the bindings keep per stream, on CPU tensors."""

from __future__ import annotations

import weakref

import pytest
import torch

from dsa_amd import _lib

CPU = torch.device("cpu")


@pytest.mark.parametrize("zeroed", [True, False])
def test_outgrown_buffers_stay_allocated(zeroed) -> None:
    """A captured graph holds the address of the buffer that it was captured with."""

    sizes, held = [], []
    for need in (1000, 5000, 5001, 70000, 200):
        ws = _lib.workspace(f"test_outgrown_{zeroed}", CPU, 0, need, zeroed=zeroed)
        assert ws.numel() >= need
        if ws.data_ptr() not in [address for address, _ in held]:
            held.append((ws.data_ptr(), weakref.ref(ws)))
            sizes.append(ws.numel())
        del ws
    assert len(held) == 4
    for address, ref in held:
        assert ref() is not None and ref().data_ptr() == address
    assert sum(sizes[:-1]) < sizes[-1]


def test_buffers_of_a_capture_are_its_own(monkeypatch) -> None:
    """The zero fill of a buffer that is made during a capture is recorded, not run,
    so that neither an eager call nor another capture may take it."""

    capture = 0
    monkeypatch.setattr(_lib, "capture_of", lambda stream: capture)

    def take(need, kind="test_capture"):
        return _lib.workspace(kind, CPU, 0, need, zeroed=True)

    eager = take(1000)
    capture = 5
    assert take(900) is eager               # fits: its fill has run
    first = take(4000)
    assert first is not eager and not first.any()
    assert take(4000) is first and take(3000) is first
    assert take(9000, "test_capture_other") is not first
    larger = take(8000)
    assert larger is not first and larger.numel() >= 8000
    capture = 6
    second = take(4000)
    assert second is not first and second is not larger
    capture = 0
    after = take(4000)
    assert all(after is not x for x in (eager, first, larger, second))
    assert take(4000) is after
    capture = 7
    assert take(4000) is after


def test_no_stream_of_the_host_is_captured() -> None:
    assert _lib.capture_of(0) == 0
