"""Executions and errors of the Python mirror, without a device: what a call waits for, and whose error it raises."""
import pytest

from _loader import load_pkg

rx = load_pkg()


class Handle:
    handle = 1


class Client:
    handle = 1

    def default_device(self):
        return Handle()


class Execution:
    """Stands for an executable of one result."""
    result_types = [((2,), "f32")]

    def __init__(self):
        self.calls = []

    def execute_sharded(self, bufs, donated=None):
        self.calls.append(bufs)
        return [rx.AsyncBuffer(Handle(), None)]


class Future:
    def __init__(self, may_fail):
        self.may_fail, self.waited = may_fail, False

    def wait(self):
        self.waited = True
        if self.may_fail:
            raise rx.ReactantInternalError("expired")


def test_a_call_raises_the_error_of_the_execution_that_made_its_argument():
    """As it did before it was used: the call itself does not run."""
    exe, fails, cannot = Execution(), Future(True), Future(False)
    call = rx.Thunk(exe, None)
    good = rx.ConcreteRArray(rx.AsyncBuffer(Handle(), cannot), (2,), "f32")
    bad = rx.ConcreteRArray(rx.AsyncBuffer(Handle(), fails), (2,), "f32")
    call(good)
    assert len(exe.calls) == 1 and not cannot.waited          # what cannot fail is not waited for
    with pytest.raises(rx.ReactantInternalError, match="expired"):
        call(good, bad, donated=[True, True])
    assert len(exe.calls) == 1 and not good.donated and not bad.donated


def test_a_call_without_results_raises_no_older_error(monkeypatch):
    exe = object.__new__(rx.LoadedExecutable)
    exe.handle, exe.client, exe.num_results, exe.waits = None, Client(), 0, False
    monkeypatch.setattr(rx, "_execute_sharded", lambda *args: None)
    rx.lib.RxExecutableNumResults(None)                         # an error that nobody asked for
    assert rx.lib.RxLastError()
    assert exe.execute_sharded([]) == []
    monkeypatch.undo()
    with pytest.raises(rx.ReactantInternalError):               # its own
        exe.execute_sharded([])
