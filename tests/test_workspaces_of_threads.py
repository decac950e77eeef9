"""Two host threads that make the first calls on a stream at once: both, and the short way from torch tensors, use one workspace (no GPU
needed: the workspaces are stand-ins)."""
from __future__ import annotations

import threading
from types import SimpleNamespace

import pytest

from asterq import linear_attention, paged_kv

MAKERS = {
    "paged attention": (paged_kv, "PagedAttentionWorkspace", "_workspaces", "_workspace"),
    "prompt and tree attention": (paged_kv, "RowsAttentionWorkspace", "_rows_workspaces", "_rows_workspace"),
    "linear attention": (linear_attention, "LinearAttentionWorkspace", "_workspaces", "_workspace"),
}


@pytest.mark.parametrize("what", MAKERS)
def test_the_short_way_keeps_the_workspace_that_lives(monkeypatch, what):
    module, cls, table, fn = MAKERS[what]
    begun, go, done = threading.Event(), threading.Event(), threading.Event()
    second, made, told = [], [], []

    class Workspace:
        nbytes = 16

        def __init__(self, device):
            made.append(self)
            self.buffer = SimpleNamespace(data_ptr=lambda: id(self))
            if threading.current_thread() in second:  # it has found none, and is overtaken
                begun.set()
                assert go.wait(20)

    class Quick:
        @staticmethod
        def workspace(kind, device, stream, ptr, nbytes):
            told.append(ptr)

    def quick():
        if threading.current_thread() not in second and not go.is_set():
            go.set()  # the other one's workspace comes now, before this one's is made known
            assert done.wait(20)
        return Quick

    monkeypatch.setattr(module, cls, Workspace)
    monkeypatch.setattr(module, table, {})
    monkeypatch.setattr(module, "_quick", quick)
    monkeypatch.setattr(module, "_capturing", lambda device: False)
    device, got = SimpleNamespace(index=0), []

    def other():
        second.append(threading.current_thread())
        got.append(getattr(module, fn)(device, 5))
        done.set()

    thread = threading.Thread(target=other)
    thread.start()
    assert begun.wait(20)
    got.append(getattr(module, fn)(device, 5))
    thread.join()
    kept = getattr(module, table)[(0, 5)]
    assert len(made) == 2 and told[-1] == id(kept)
    assert got == [kept, kept]
    assert getattr(module, fn)(device, 5) is kept
