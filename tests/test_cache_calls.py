"""What the cache calls' Python side does before the library is called, with
stand-ins for torch and its tensors: no device is needed."""
import sys
import threading
import types

import pytest

from gopherllm_amd import api


class Torch(types.SimpleNamespace):
    """torch as _here uses it; `slow` is called in the middle of the first look at it."""

    def __init__(self, slow=lambda: None):
        super().__init__(float32="float32", uint8="uint8", int8="int8", uint32="uint32", int16="int16", uint16="uint16", slow=slow,
                         cuda=types.SimpleNamespace(current_device=lambda: 0),
                         _C=types.SimpleNamespace(_cuda_getCurrentRawStream=lambda at: 77))

    @property
    def int32(self):
        self.slow()
        return "int32"


@pytest.fixture
def fresh(monkeypatch):
    """api as it is before its first call; returns the way to give it a torch."""
    monkeypatch.setattr(api, "_kinds", {})
    for name in ("_torch", "_raw_stream"):
        monkeypatch.setattr(api, name, None, raising=False)
        monkeypatch.delattr(api, name)

    def give(torch):
        monkeypatch.setitem(sys.modules, "torch", torch)
        return torch
    return give


def test_first_calls_of_two_threads(fresh):
    """A second thread's first call while the first thread's is half way through its setup."""
    inside, go = threading.Event(), threading.Event()

    def slow():
        if not inside.is_set():
            inside.set()
            assert go.wait(20)

    fresh(Torch(slow))
    got = []
    first = threading.Thread(target=lambda: got.append(api._here()))
    first.start()
    try:
        assert inside.wait(20)
        assert api._here() == (0, 77)
        assert set(api._kinds) == set(api._DTYPES)
    finally:
        go.set()
        first.join()
    assert got == [(0, 77)]
