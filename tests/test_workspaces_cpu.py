"""The cached workspaces of ``ops``: what a captured graph holds stays its own. Streams and captures are stand-ins, so that this runs without a GPU."""

import weakref

import pytest
import torch

from cleave_b200 import ops


@pytest.fixture
def host(monkeypatch):
    """Workspaces in host memory; ``host["stream"]`` and ``host["capturing"]`` are what the calls see."""
    state = {"stream": 1, "capturing": False}
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_outgrown", [], raising=False)
    monkeypatch.setattr(ops, "_stream", lambda: state["stream"])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    return state


def test_a_workspace_is_kept_per_kind_and_stream(host):
    a = ops.workspace("a", 1000, "cpu")
    assert a.numel() >= 1000 and not a.any()
    assert ops.workspace("a", 500, "cpu") is a and ops.workspace("b", 500, "cpu") is not a
    host["stream"] = 2
    assert ops.workspace("a", 500, "cpu") is not a


def test_an_outgrown_workspace_is_not_given_away(host):
    """A graph captured with the smaller one replays kernels that count in it."""
    alive = []
    for n in (1000, 2000, 5000, 5001, 70000):
        ws = ops.workspace("a", n, "cpu")
        assert ws.numel() >= n
        alive.append(weakref.ref(ws))
    del ws
    assert all(r() is not None for r in alive)


def test_outgrown_workspaces_are_smaller_than_the_one_in_use(host):
    for n in range(1000, 100000, 777):
        ws = ops.workspace("a", n, "cpu")
    assert sum(t.numel() for t in ops._outgrown) < ws.numel() < 2 * 100000


def test_a_workspace_made_under_capture_stays_with_captures(host):
    """It lies in the graph's pool and is zero-filled by the graph alone, when that is replayed."""
    host["capturing"] = True
    captured = ops.workspace("a", 1000, "cpu")
    assert ops.workspace("a", 1000, "cpu") is captured
    host["capturing"] = False
    eager = ops.workspace("a", 1000, "cpu")
    assert eager is not captured
    host["capturing"] = True
    assert ops.workspace("a", 1000, "cpu") is eager  # one that is zero already serves a capture too
    larger = ops.workspace("a", 5000, "cpu")
    host["capturing"] = False
    assert ops.workspace("a", 1000, "cpu") is eager and ops.workspace("a", 5000, "cpu") is not larger
