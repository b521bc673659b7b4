"""The garbage collector waits until the last of the captures that are on at the same time has ended (no GPU: a runtime that
records nothing)."""
import gc
import threading

import pytest

from test_abi import tsk  # noqa: F401  (fixture)


class Runtime:
    def __getattr__(self, name):
        return lambda *a: 0


class Stream:
    h = None


@pytest.fixture
def graph(tsk, monkeypatch):  # noqa: F811
    monkeypatch.setattr(tsk, "hip", lambda: Runtime())
    assert gc.isenabled()
    yield tsk.Graph
    gc.enable()


@pytest.mark.parametrize("first_in_first_out", [True, False])
def test_two_threads(graph, first_in_first_out):
    began, go_on, seen = [threading.Event(), threading.Event()], [threading.Event(), threading.Event()], []

    def work(i):
        began[i].set()
        assert go_on[i].wait(20)
        seen.append(gc.isenabled())

    threads = [threading.Thread(target=graph, args=(Stream(), lambda i=i: work(i))) for i in range(2)]
    for i in range(2):
        threads[i].start()
        assert began[i].wait(20)
    for i in (0, 1) if first_in_first_out else (1, 0):
        assert not gc.isenabled()
        go_on[i].set()
        threads[i].join(20)
        assert not threads[i].is_alive()
    assert seen == [False, False] and gc.isenabled()


def test_a_capture_that_fails(graph):
    def fail():
        raise RuntimeError("no")

    def outer():
        with pytest.raises(RuntimeError):
            graph(Stream(), fail)
        assert not gc.isenabled()

    graph(Stream(), outer)
    assert gc.isenabled()


def test_a_collector_that_was_off_stays_off(graph):
    gc.disable()
    graph(Stream(), lambda: graph(Stream(), lambda: None))
    assert not gc.isenabled()
