"""Which memory the layers' default workspaces are, without a GPU."""
import gc
import threading

import pytest
import torch

from exq_amd import _lib

CPU = torch.device("cpu", 0)


@pytest.fixture(autouse=True)
def _clear():
    _lib.clear_workspace_cache()
    yield
    _lib.clear_workspace_cache()


def _in_thread(fn):
    got = []
    t = threading.Thread(target=lambda: got.append(fn()))
    t.start()
    t.join()
    return got[0]


def test_a_stream_keeps_its_workspace_and_kinds_are_apart():
    a = _lib.workspace(CPU, 100, "fused", 7)
    assert _lib.workspace(CPU, 100, "fused", 7) is a
    others = [_lib.workspace(CPU, 100, "fused", 8), _lib.workspace(CPU, 100, "mxfp4", 7)]
    assert len({t.data_ptr() for t in (a, *others)}) == 3
    more = _lib.workspace(CPU, a.numel() + 1, "fused", 7)
    assert more.numel() > a.numel() and _lib.workspace(CPU, 100, "fused", 7) is more


@pytest.mark.parametrize("kind", ["fused", "scratch", "mxfp4"])
def test_threads_on_one_stream_have_a_workspace_each(kind):
    """A layer is several launches that hand their results over in the workspace, and two
    threads' launches on one stream come in any order."""
    mine = _lib.workspace(CPU, 100, kind, 7)
    here, go = threading.Barrier(3), threading.Event()
    theirs = []

    def work():
        theirs.append(_lib.workspace(CPU, 100, kind, 7))
        here.wait(10)
        go.wait(10)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    here.wait(10)
    assert len({t.data_ptr() for t in (mine, *theirs)}) == 3
    go.set()
    for t in threads:
        t.join()
    assert _lib.workspace(CPU, 100, kind, 7) is mine


def test_a_thread_takes_its_workspaces_with_it():
    gc.collect()
    _lib.workspace(CPU, 100, "fused", 7)
    before = len(_lib._all_buffers)
    _in_thread(lambda: _lib.workspace(CPU, 100, "fused", 7).numel())
    gc.collect()
    assert len(_lib._all_buffers) == before


def test_clearing_reaches_every_thread():
    mine = _lib.workspace(CPU, 100, "fused", 7)
    _in_thread(_lib.clear_workspace_cache)
    assert _lib.workspace(CPU, 100, "fused", 7) is not mine


def test_a_graph_has_workspaces_of_its_own(monkeypatch):
    """Two graphs captured on one stream may run at once, and a buffer whose address a graph
    holds must not be let go of when a later call needs a larger one."""
    eager = _lib.workspace(CPU, 100, "fused", 7)
    monkeypatch.setattr(_lib, "_capturing", lambda device: True)
    graphs = [_lib.workspace(CPU, 100, "fused", 7) for _ in range(2)]
    assert len({t.data_ptr() for t in (eager, *graphs)}) == 3
    monkeypatch.undo()
    assert _lib.workspace(CPU, 100, "fused", 7) is eager
