"""What the cache calls' Python side does before the library is called, with
stand-ins for torch and its tensors: no device is needed."""
import ctypes as C
import sys
import threading
import types

import pytest

import gopherllm_amd as g
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


# --- a layer's rows as tensors -------------------------------------------------


class Cache(C.Structure):
    """csrc/kv_cache.h"""
    _fields_ = [(n, C.c_int) for n in ("layers", "kv_dim_k", "kv_dim_v", "max_len")] + [
        ("k", C.c_void_p), ("v", C.c_void_p), ("device", C.c_int)]


def cache(device=0, layers=2, kd=256, vd=128, rows=100):
    """A KVCacheF16 over a handle of our own; its rows' addresses are never read."""
    at = (C.c_void_p * (2 * layers))(*[4096 * (i + 1) for i in range(2 * layers)])
    raw = Cache(layers, kd, vd, rows, C.addressof(at), C.addressof(at) + 8 * layers, device)
    kv = api.KVCacheF16(layers, kd, vd, rows, handle=C.addressof(raw), owned=False)
    kv.kept = (at, raw)
    return kv


@pytest.mark.parametrize("device", [0, 3])
def test_tensors_are_on_the_caches_device(monkeypatch, device):
    """Whatever the current device is: torch copies rows that are asked for on another one."""
    import torch
    asked = []
    monkeypatch.setattr(torch, "as_tensor", lambda rows, device: asked.append((rows.__cuda_array_interface__, str(torch.device(device)))))
    cache(device).tensors(1)
    assert [(a["data"][0], a["shape"], d) for a, d in asked] == [(8192, (100, 256), f"cuda:{device}"), (16384, (100, 128), f"cuda:{device}")]


def test_tensors_refusals():
    kv = cache()
    for layer in (-1, 2):
        with pytest.raises(ValueError):
            kv.tensors(layer)
    kv.release()
    with pytest.raises(ValueError, match="released"):
        kv.tensors(0)
    assert g.load().gllm_hip_kv_device(None) == g.EINVAL
