"""What the cache calls' Python side does before the library is called, with
stand-ins for torch and its tensors: no device is needed."""
import ctypes as C
import sys
import threading
import types

import numpy as np
import pytest

import gopherllm_amd as g
from gopherllm_amd import _lib, api


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


# --- sizes and strides past 32 bits, which ctypes would cut ----------------------


class Tensor:
    """A device tensor as the calls look at it: shape and strides without memory."""

    def __init__(self, *shape, kind="float32", strides=None, device=0):
        self.shape, self.dtype, self.device, self.is_cuda = shape, kind, device, True
        self.strides = strides or [int(np.prod(shape[i + 1:], dtype=np.int64)) for i in range(len(shape))]
        self.whole = strides is None

    def stride(self, i):
        return self.strides[i]

    def get_device(self):
        return self.device

    def numel(self):
        return int(np.prod(self.shape, dtype=np.int64))

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return self.whole

    def data_ptr(self):
        return 4096


def ints(*shape):
    return Tensor(*shape, kind="int32")


@pytest.fixture
def calls(fresh, monkeypatch):
    """The library calls that get through, with their arguments."""
    fresh(Torch())
    got = []
    monkeypatch.setattr(api, "call", lambda name, *args: got.append((name, *args)))
    return got


def rope(hd=64):
    r = object.__new__(api.Rope)
    r.handle, r.head_dim = None, hd
    return r


FAR = (1 << 32) + 128  # 128 when it is cut
SHARED = dict(layer=0, q=Tensor(3, 512), n_heads=8, n_kv_heads=2, hd=64, start=0, length=10, starts=ints(3), lens=ints(3), most=4,
              scale=0.1, out=Tensor(3, 512))
MASS = dict(layer=0, q=Tensor(3, 512), n_heads=8, n_kv_heads=2, hd=64, start=0, end=9, scale=0.1, mass=Tensor(2, 100), out=Tensor(3, 512))
KEEP = dict(n_kv_heads=2, hd=64, length=50, budget=20, mass=Tensor(2, 2, 100), pos=ints(2, 2, 100), mass_out=Tensor(2, 2, 30),
            pos_out=ints(2, 2, 30), now=50)
EVICT = dict(layer=0, n_kv_heads=2, hd=64, k=Tensor(128), v=Tensor(128), start=0, length=50, mass=Tensor(2, 100), pos=ints(2, 100), now=ints(1))


@pytest.mark.parametrize("name,args,changed", [("attend_shared_dev", SHARED, dict(a)) for a in [
    dict(layer=FAR), dict(start=FAR), dict(length=FAR), dict(most=FAR), dict(start=-FAR), dict(length=-(1 << 32))]] +
    [("attend_mass_dev", MASS, dict(a)) for a in [dict(start=FAR), dict(end=FAR), dict(layer=FAR), dict(mass=Tensor(2, FAR))]] +
    [("keep_dev", KEEP, dict(a)) for a in [
        dict(length=FAR), dict(budget=FAR), dict(now=FAR), dict(sinks=1 << 32), dict(recent=1 << 40), dict(start=FAR), dict(dst_start=FAR),
        dict(mass=Tensor(2, 2, FAR), pos=None), dict(mass_out=Tensor(2, 2, FAR), pos_out=ints(2, 2, FAR))]] +
    [("evict_store_dev", EVICT, dict(a)) for a in [
        dict(length=FAR), dict(sinks=1 << 32), dict(recent=1 << 40), dict(start=FAR), dict(layer=FAR),
        dict(mass=Tensor(2, FAR), pos=ints(2, FAR))]])
def test_sizes_past_32_bits_are_refused(calls, name, args, changed):
    kv = cache()
    lead = (cache(rows=30),) if name == "keep_dev" else ()
    getattr(kv, name)(*lead, **args)
    assert len(calls) == 1  # as it is, the call gets through
    with pytest.raises(ValueError):
        getattr(kv, name)(*lead, **{**args, **changed})
    assert len(calls) == 1


def test_a_layer_past_32_bits_is_refused(calls):
    args = dict(rope=rope(), q=None, k=Tensor(3, 128), v=Tensor(3, 128), positions=ints(3), rows=ints(3))
    with pytest.raises(ValueError, match="32"):
        cache().store_rope_dev(1 << 32, **args)
    assert not calls


def test_negative_sizes_are_the_librarys_to_refuse(calls):
    cache().attend_shared_dev(**{**SHARED, "start": -1, "length": -5})
    assert calls[0][8:10] == (-1, -5)


@pytest.mark.parametrize("which", ["q", "k", "v", "q_out"])
def test_row_strides_past_32_bits_are_refused(calls, which):
    kv, n, d = cache(), 3, 128
    args = dict(q=Tensor(n, d), k=Tensor(n, d), v=Tensor(n, d), positions=ints(n), rows=ints(n), q_out=Tensor(n, d))
    wide = {**args, which: Tensor(n, d, strides=[(1 << 31) - 1, 1])}
    kv.store_rope_dev(0, rope(), **wide)
    assert len(calls) == 1 and (1 << 31) - 1 in calls[0]
    for stride in (1 << 31, FAR):
        with pytest.raises(ValueError, match="32"):
            kv.store_rope_dev(0, rope(), **{**args, which: Tensor(n, d, strides=[stride, 1])})
        with pytest.raises(ValueError, match="32"):
            rope().apply_dev(Tensor(n, d, strides=[stride, 1]), ints(n), Tensor(n, d))
    assert len(calls) == 1


def test_more_tokens_than_32_bits_count_are_refused(calls):
    n = (1 << 32) + 1
    with pytest.raises(ValueError, match="32"):
        rope().apply_dev(Tensor(n, 128), ints(n), Tensor(n, 128))
    with pytest.raises(ValueError, match="32"):
        cache().attend_shared_dev(**{**SHARED, "q": Tensor(n, 512), "out": Tensor(n, 512), "starts": ints(n), "lens": ints(n)})
    assert not calls


@pytest.mark.parametrize("kw", [dict(head_dim=FAR), dict(head_dim=128, rot_dim=FAR), dict(head_dim=128, orig_ctx=FAR)])
def test_rope_sizes_past_32_bits_are_refused(kw):
    with pytest.raises(ValueError, match="32"):
        g.Rope.config(**kw)


@pytest.mark.parametrize("name,args", [("attend_shared_bytes", (4, 8, 2, 64, FAR, 4)), ("attend_shared_bytes", (4, 8, 2, 64, 10, FAR)),
                                       ("attend_mass_bytes", (4, 8, 2, 64, FAR)), ("keep_bytes", (4, 8, FAR))])
def test_workspaces_past_32_bits_are_refused(name, args):
    with pytest.raises(ValueError, match="32"):
        getattr(g, name)(*args)


# --- rows of another width ----------------------------------------------------


@pytest.mark.parametrize("name,args", [("attend_shared_dev", SHARED), ("attend_mass_dev", MASS)])
def test_rows_of_another_width_are_refused(calls, name, args):
    """Tokens are read and written n_heads * hd apart: wider rows, such as a fused projection's, are not."""
    kv = cache()
    for wrong in (dict(q=Tensor(3, 768)), dict(q=Tensor(3, 2, 512)), dict(out=Tensor(3, 768)), dict(out=Tensor(4, 520)), dict(out=Tensor(3, 511))):
        with pytest.raises(ValueError):
            getattr(kv, name)(**{**args, **wrong})
    assert not calls
    right = [dict(q=Tensor(3, 8, 64)), dict(out=Tensor(3, 8, 64)), dict(out=Tensor(5, 512)), dict(out=Tensor(4000)), dict(out=Tensor(24, 64))]
    if name == "attend_shared_dev":
        right.append(dict(q=Tensor(512), starts=ints(1), lens=ints(1), out=Tensor(8, 64)))
    for also in right:
        getattr(kv, name)(**{**args, **also})
    assert len(calls) == len(right)


# --- workspaces -----------------------------------------------------------------


def test_no_workspace_for_sizes_that_a_call_refuses():
    """Longer than a cache can be, and head sizes that attention does not take."""
    far = 1 << 30
    for n_kv in (1, 512, 4096):
        assert g.attend_shared_bytes(1, n_kv, n_kv, 8, far, 0) > 0 and g.attend_mass_bytes(1, n_kv, n_kv, 8, far) >= 4 * n_kv * far
        for length in (far + 1, 2**31 - 1):
            assert g.attend_shared_bytes(1, n_kv, n_kv, 8, length, 0) == 0 and g.attend_mass_bytes(1, n_kv, n_kv, 8, length) == 0
    for hd in (0, 1, 7, 12, 127, 136):
        assert g.attend_shared_bytes(2, 4, 2, hd, 10, 3) == 0 and g.attend_mass_bytes(2, 4, 2, hd, 10) == 0
    assert g.attend_shared_bytes(2, 4, 2, 64, 10, 2**31 - 1) > 0  # a plan longer than any cache is still one


HEADS = [(32, 8, 128), (8, 2, 64), (40, 8, 80), (71, 1, 128), (16, 16, 8), (3, 1, 24)]


@pytest.mark.parametrize("heads,n_kv,hd", HEADS)
def test_workspaces_never_fall(heads, n_kv, hd):
    """One workspace, sized for the most tokens and the longest ranges, serves every smaller call."""
    ns = [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 63, 64, 65, 128, 256, 300, 1024, 4096]
    lens = [0, 1, 31, 127, 128, 129, 300, 640, 1000, 2049, 4001, 4096, 5000, 8192, 8193, 16001, 32768, 50000, 131072, 1 << 20, 1 << 30]
    mosts = [0, 1, 17, 128, 129, 640, 1024, 4096, 8193, 1 << 20, 2**31 - 1]
    size = {(n, a, b): g.attend_shared_bytes(n, heads, n_kv, hd, a, b) for n in ns for a in lens for b in mosts}
    for (n, a, b), x in size.items():
        for other in ((m, a, b) for m in ns[:ns.index(n)][-1:]), ((n, m, b) for m in lens[:lens.index(a)][-1:]), ((n, a, m) for m in mosts[:mosts.index(b)][-1:]):
            for o in other:
                assert size[o] <= x, (o, (n, a, b))
    mass = {(n, a): g.attend_mass_bytes(n, heads, n_kv, hd, a) for n in ns for a in lens if n <= a}
    for (n, a), x in mass.items():
        assert all(mass[n, m] <= x for m in lens if n <= m < a), (n, a)
        assert all(mass[m, a] <= x for m in ns if m < n), (n, a)
    # and they stay within twice the partial results of the largest grid
    assert size[64, 32768, 1024] <= 4 * (2 + hd) * 2 * (64 * heads + 65536 + 512 * heads // n_kv) + 256
    assert [g.keep_bytes(3, n_kv, b) for b in (1, 5, 700)] == sorted(g.keep_bytes(3, n_kv, b) for b in (1, 5, 700))


def test_every_length_fits_the_longest_ones_workspace():
    for n, most in ((1, 0), (8, 640), (33, 200), (64, 1024)):
        sizes = [g.attend_shared_bytes(n, 32, 8, 128, length, most) for length in range(0, 9000, 7)]
        assert sizes == sorted(sizes)
        sizes = [g.attend_mass_bytes(n, 32, 8, 128, length) for length in range(n, 9000, 7)]
        assert sizes == sorted(sizes)


def test_an_empty_workspace_is_refused(calls):
    """Its null address would stand for the library's own scratch, which graphs share."""
    class Empty(Tensor):
        def data_ptr(self):
            return 0

    for name, args in (("attend_shared_dev", SHARED), ("attend_mass_dev", MASS), ("keep_dev", KEEP)):
        lead = (cache(rows=30),) if name == "keep_dev" else ()
        with pytest.raises(ValueError, match="work"):
            getattr(cache(), name)(*lead, **args, work=Empty(0, kind="uint8"))
        assert not calls
        getattr(cache(), name)(*lead, **args, work=Tensor(64, kind="uint8"))
        assert calls.pop()[-3:] == (4096, 64, 77)


P = 1 << 24  # addresses that are never read: 2 layers x 2 heads x 100 rows of mass from here on


@pytest.mark.parametrize("at", [P, P + 1596, P + (1 << 20) + 1584, P + (2 << 20) - 304, P + (2 << 20), P + (3 << 20), P + (3 << 20) + 464])
def test_keep_refuses_a_workspace_over_its_tensors(at):
    """The workspace holds the rows to copy: written over, they would be any rows."""
    src, dst = cache(), cache(rows=30)
    mass, pos, mass_out, pos_out = (C.c_void_p(P + (i << 20)) for i in range(4))
    size = g.keep_bytes(2, 2, 20)
    at = at // 16 * 16
    rc = g.load().gllm_hip_kv_keep_dev(C.c_void_p(src.handle), C.c_void_p(dst.handle), 2, 64, 0, 50, 0, 20, 1, 2, 50, mass, pos, 100, mass_out,
                                       pos_out, 30, C.c_void_p(at), size, None)
    assert rc == g.EINVAL and "overlaps" in _lib.last_error()


def test_keep_takes_a_workspace_next_to_its_tensors():
    """Refused for want of a device only, not for its place."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device would run it")
    src, dst = cache(), cache(rows=30)
    mass, pos, mass_out, pos_out = (C.c_void_p(P + (i << 20)) for i in range(4))
    for at in (P - 320, P + 1600, P + (2 << 20) - 320, P + (3 << 20) + 480):
        rc = g.load().gllm_hip_kv_keep_dev(C.c_void_p(src.handle), C.c_void_p(dst.handle), 2, 64, 0, 50, 0, 20, 1, 2, 50, mass, pos, 100, mass_out,
                                           pos_out, 30, C.c_void_p(at), g.keep_bytes(2, 2, 20), None)
        assert rc != g.OK and "overlap" not in _lib.last_error()
