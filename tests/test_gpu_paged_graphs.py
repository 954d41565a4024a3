"""Captured calls of the paged cache's operators beside eager ones on the capturing
stream.  Every replay is compared with the eager result, bit for bit."""

from __future__ import annotations

import pytest
import torch

from dsa_amd import _lib, paged
from test_gpu_paged import BF16, FP8, Case

pytestmark = pytest.mark.gpu


def _decode(device, seed, dtype=BF16):
    c = Case(device, seed, [3000, 700], [1, 1], 8, 2, 128, 16, dtype)
    args = (c.q.to(device), c.cache, *c.device_args(starts=False))
    lists = torch.arange(1500, device=device).expand(2, 1500).contiguous()

    def step():
        return paged.attention(*args), paged.selected_attention(*args[:4], lists)

    return step


def _prompt(device, seed, tokens):
    c = Case(device, seed, [4000], [tokens], 16, 2, 128, 16, BF16)
    args = (c.q.to(device), c.cache, *c.device_args(starts=False))
    return lambda: paged.attention(*args)


def _same(got, want) -> bool:
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_a_larger_call_after_the_capture(device, dtype) -> None:
    """A captured decode step, then a prompt on the same stream, whose workspace is
    larger, and other tensors where the step's may have been."""

    step, prompt = _decode(device, 1, dtype), _prompt(device, 2, 300)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        want = step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
        large = prompt()
        junk = [torch.full((1 << n,), 77, dtype=torch.uint8, device=device) for n in range(20, 26) for _ in range(3)]
        for _ in range(4):
            for x in got:
                x.zero_()
            graph.replay()
            stream.synchronize()
            assert _same(got, want)
            assert torch.equal(prompt(), large)
        stream.synchronize()
        assert all(bool((x == 77).all()) for x in junk)


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 2, 0)])
def test_captures_without_a_call_before_on_their_stream(device, order) -> None:
    """Three graphs of growing workspaces, captured on a stream that no call has run
    on, replayed in any order, with eager calls on that stream before the first."""

    calls = [_decode(device, 3), _decode(device, 4, FP8), _prompt(device, 5, 300)]
    want = [call() for call in calls]                     # on another stream
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs, got = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            got.append(call())
    torch.cuda.synchronize()

    def same(i, out):
        return torch.equal(out, want[i]) if torch.is_tensor(out) else _same(out, want[i])

    with torch.cuda.stream(stream):
        assert same(0, calls[0]())
    for turn in range(3):
        for i in order:
            for x in (got[i],) if torch.is_tensor(got[i]) else got[i]:
                x.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert same(i, got[i]), (turn, i)
        with torch.cuda.stream(stream):
            assert same(2, calls[2]()) and same(1, calls[1]())
        torch.cuda.synchronize()


def test_captures_have_ids_of_their_own(device) -> None:
    stream = torch.cuda.Stream()
    x = torch.zeros(4, device=device)
    ids = []
    for _ in range(3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x += 1
            ids.append(_lib.capture_of(stream.cuda_stream))
        assert _lib.capture_of(stream.cuda_stream) == 0
        graph.replay()
    torch.cuda.synchronize()
    assert len(set(ids)) == 3 and 0 not in ids
    assert x.tolist() == [3.0] * 4
