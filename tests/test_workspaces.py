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
