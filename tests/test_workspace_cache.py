"""The cached workspaces: a graph keeps the addresses that its capture saw, so a capture shares none
with calls outside it or with another capture.  CPU only (host tensors stand in for device memory)."""

from __future__ import annotations

import types

import pytest
import torch


@pytest.fixture
def host(monkeypatch):
    """ops with an empty cache, one stream, and a capture number that the test sets."""
    from dels_b200 import ops

    state = {"capture": 0}
    monkeypatch.setattr(ops, "_ws_cache", {})
    monkeypatch.setattr(ops, "_capture_ws", {}, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(ops, "_capture_id", lambda stream: state["capture"], raising=False)
    return ops, state, torch.device("cpu")


def test_captures_share_no_workspace(host):
    ops, state, dev = host
    eager = ops._stream_workspace(1000, dev, 7)
    seen = [eager]
    for capture in (11, 12):
        state["capture"] = capture
        ws = ops._stream_workspace(1000, dev, 7)
        assert all(ws is not other for other in seen)
        assert ops._stream_workspace(500, dev, 7) is ws  # one for all calls of the capture
        assert ops.workspace(500, dev) is ws
        seen.append(ws)
    state["capture"] = 0
    assert ops._stream_workspace(1000, dev, 7) is eager


def test_growth_outside_a_capture_leaves_the_captures_alone(host):
    ops, state, dev = host
    state["capture"] = 3
    small = ops._stream_workspace(1000, dev, 7)
    large = ops._stream_workspace(3 << 20, dev, 7)
    assert large is not small and large.nbytes >= 3 << 20
    assert ops._stream_workspace(1000, dev, 7) is large
    state["capture"] = 0
    grown = ops._stream_workspace(5 << 20, dev, 7)
    assert grown is not large and ops._stream_workspace(1000, dev, 7) is grown
    state["capture"] = 3
    assert ops._stream_workspace(1000, dev, 7) is large
