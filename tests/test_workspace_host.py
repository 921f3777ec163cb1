"""The per-stream workspaces' bookkeeping, on host tensors with the device calls left out."""
import gc
import weakref

import pytest
import torch

from next_step_ai_amd import _lib, _runtime


@pytest.fixture()
def streams(monkeypatch):
    """A current stream that a test sets; the calls that would go to the device, listed."""
    class Now:
        handle, capturing, calls = 7, False, []

    now = Now()
    now.calls = []
    monkeypatch.setattr(_runtime, "stream_handle", lambda device: now.handle)
    monkeypatch.setattr(_runtime, "_workspaces", {})
    monkeypatch.setattr(_lib, "call", lambda name, *args: now.calls.append((name, *args)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capturing)
    return now


def test_a_workspace_that_has_grown_keeps_the_old_memory(streams):
    """A captured graph holds the address of the workspace that it was recorded with, and nothing else of it: the memory
    stays when a later call on the stream needs a larger one."""
    cpu = torch.device("cpu")
    first = _runtime.workspace(100, cpu)
    assert first.numel() == 1 << 20 and first.data_ptr() % 256 == 0
    assert _runtime.workspace(1 << 20, cpu) is first
    address, alive = first.data_ptr(), weakref.ref(first)
    del first
    second = _runtime.workspace((1 << 20) + 1, cpu)
    assert second.numel() == 2 << 20 and second.data_ptr() != address
    gc.collect()
    assert alive() is not None and alive().data_ptr() == address
    assert _runtime.workspace(1, cpu) is second
    assert [c[0] for c in streams.calls] == ["nsmlp_workspace_init"] * 2
    streams.handle = 8
    assert _runtime.workspace(1, cpu) is not second


def test_a_workspace_made_inside_a_capture_is_the_graphs_alone(streams):
    """Its counters are cleared by a node of the graph, so nobody else may use it before the graph has run."""
    cpu = torch.device("cpu")
    streams.capturing = True
    captured = _runtime.workspace(100, cpu)
    again = _runtime.workspace(100, cpu)  # the next call of the same capture
    assert again is not captured and [c[0] for c in streams.calls] == ["nsmlp_workspace_init"] * 2
    streams.capturing = False
    eager = _runtime.workspace(100, cpu)
    assert eager is not captured and len(streams.calls) == 3 and streams.calls[2][1] == eager.data_ptr()
    streams.capturing = True
    assert _runtime.workspace(100, cpu) is eager  # one that the stream had before is used as it is
    larger = _runtime.workspace(eager.numel() + 1, cpu)
    streams.capturing = False
    assert larger is not eager and _runtime.workspace(100, cpu) is eager
