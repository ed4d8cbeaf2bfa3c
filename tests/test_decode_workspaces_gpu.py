"""Workspaces of the decode kernels: grown, captured, abandoned, of many streams."""

from __future__ import annotations

import pytest
import torch

from test_cache8_decode_gpu import INT8, _case
from vllm_mps_b200 import kernels as K

pytestmark = pytest.mark.gpu


def _small(seed=1):
    return _case([3000, 17], 8, 2, 64, torch.float16, INT8, seed)


def _large(seed=2):
    return _case([2000, 900], 32, 2, 128, torch.bfloat16, INT8, seed)


def _capture(c, ws):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.paged_decode_attention_cache8(**c, workspace=ws)
    return graph, out


def test_outgrown_buffers_stay_for_the_graphs_that_use_them():
    small, large, ws = _small(), _large(), K.DecodeWorkspace()
    want = K.paged_decode_attention_cache8(**small, workspace=ws)
    first = next(iter(ws._buf.values()))
    graph, out = _capture(small, ws)
    K.paged_decode_attention_cache8(**large, workspace=ws)
    assert next(iter(ws._buf.values())).numel() > first.numel() and ws._outgrown[0] is first
    # What would be handed out in its place is not written to.
    others = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in [first.numel()] * 4]
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert all((t == 7).all() for t in others)


def test_a_capture_before_any_call():
    """The graph has a buffer of its own; the workspace is as it was."""
    small, ws = _small(), K.DecodeWorkspace()
    want = K.paged_decode_attention_cache8(**small)
    torch.cuda.synchronize()
    graph, out = _capture(small, ws)
    assert not ws._buf
    assert torch.equal(K.paged_decode_attention_cache8(**small, workspace=ws), want)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_counters_are_zeroed_after_a_wait_that_gave_up(monkeypatch):
    """A call that gave up leaves counters above zero (put there here by hand)."""
    class GaveUp:
        def vmps_debug_error_word(self, stream, word):
            word._obj.value = 8
            return 0

    c, ws = _small(), K.DecodeWorkspace()
    want = K.paged_decode_attention_cache8(**c, workspace=ws)
    K.paged_decode_attention_cache8(**c)
    for buf in (*ws._buf.values(), *K._cache8_buffers.values()):
        buf[:K._CACHE8_COUNTER_BYTES] = 1
    with monkeypatch.context() as m:
        m.setattr(K, "load_library", GaveUp)
        assert K.error_word() == 8
    assert torch.equal(K.paged_decode_attention_cache8(**c, workspace=ws), want)
    assert torch.equal(K.paged_decode_attention_cache8(**c), want)


def test_many_streams(monkeypatch):
    monkeypatch.setattr(K, "_CACHE8_STREAMS", 3)
    cases = [_small(seed) for seed in range(6)]
    want = [K.paged_decode_attention_cache8(**c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(K.paged_decode_attention_cache8(**c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    assert len(K._cache8_buffers) <= 3
