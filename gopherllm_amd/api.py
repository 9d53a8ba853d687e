"""Python mirror of the reference's matvec / attention call surface over the
C ABI (include/gllm_hip.h).  Names follow the Go API they stand in for:

    Weight.matvec_into       (Weight).MatvecInto        model.go:670
    Weight.argmax_matvec     (Weight).ArgmaxMatvec      model.go:754
    matvec_q4k_into          MatvecQ4KInto              simd.go:261
    matvec_q6k_into          MatvecQ6KInto              simd.go:413
    matvec_q8_0_into         MatvecQ8_0Into             simd.go:204
    matvec2_into / matvec3_into   MatvecQ4K2IntoWithXSums simd.go:295,
                             Q4KMatvec3IntoWithXSums    metal.go:14
    matvec_batch             matvecBatchQ8              kernels_amd64.go:470
    Weight.rows_dev          (Weight).RowInto           model.go:1034
    KVCacheF16.store_kv      (*KVCache).storeKV         model.go:1466
    KVCacheF16.attend_head_group (*KVCache).attendHeadGroup model.go:1516
    Rope, KVCacheF16.store_rope_dev  prepareRopeScratch / applyPreparedRope model.go:3020-3093

Host arrays are numpy; device arrays are torch tensors on a ROCm device (torch
supplies device memory and streams only -- every computation is a HIP kernel
of libgllm_hip).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import (TYPE_Q4_K, TYPE_Q6_K, TYPE_Q8_0, ATTN_EXACT, ATTN_SPLITK, call, call_ptr,
                   load)



def row_bytes(qtype: int, cols: int) -> int:
    """GGMLType.DataSize for one row (gguf.go:241-297)."""
    return int(load().gllm_hip_ggml_data_size(int(qtype), int(cols)))


def _np_ptr(a):
    return a.ctypes.data_as(C.c_void_p)


def _dev_ptr(t):
    return C.c_void_p(t.data_ptr())


_DTYPES = {"f32": ("float32",), "u8": ("uint8", "int8"), "u32": ("int32", "uint32"),
           "i32": ("int32",), "u16": ("int16", "uint16")}


def _dev(t, kind: str, numel: int, what: str):
    """Device pointer of tensor t after checking that it is a contiguous
    device tensor of the element kind with at least numel elements: a wrong
    tensor would otherwise become an out-of-bounds device access."""
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{what}: expected a device tensor")
    if str(t.dtype).replace("torch.", "") not in _DTYPES[kind]:
        raise ValueError(f"{what}: dtype {t.dtype}, expected {kind}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: tensor must be contiguous")
    if t.numel() < numel:
        raise ValueError(f"{what}: {t.numel()} elements, need at least {numel}")
    return _dev_ptr(t)


def _host_f32(a, numel: int, what: str):
    a = np.ascontiguousarray(a, dtype=np.float32)
    if a.size < numel:
        raise ValueError(f"{what}: {a.size} elements, need at least {numel}")
    return a


_kinds = {}


def _here():
    """(current device, its current stream) for the calls that check their
    tensors' device.  A decode step makes a few such calls per layer, each a few
    microseconds on the GPU, so they look torch up once and ask it for plain
    numbers (a torch Stream object alone is 3 us)."""
    global _kinds, _torch, _raw_stream
    if not _kinds:
        import torch
        kinds = {kind: frozenset(getattr(torch, n) for n in names if hasattr(torch, n)) for kind, names in _DTYPES.items()}
        _torch = torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda at: torch.cuda.current_stream(at).cuda_stream)
        _kinds = kinds  # last and whole: another thread that sees it sees the others
    at = _torch.cuda.current_device()
    return at, _raw_stream(at)


def _ptr(t, kind: str, numel: int, what: str, at: int):
    """_dev's pointer of a tensor that has to be on device `at` as well."""
    if t.dtype in _kinds[kind] and t.get_device() == at and t.numel() >= numel and t.is_contiguous():
        return t.data_ptr()
    _dev(t, kind, numel, what)
    raise ValueError(f"{what}: on device {t.get_device()}, the current one is {at}")


def _ptr_rows(t, kind: str, n: int, dim: int, what: str, at: int):
    """(pointer, row stride) of n rows of dim values: a 1-D tensor of one row, or
    a 2-D tensor whose rows are contiguous and may be apart."""
    if t.get_device() < 0:
        raise ValueError(f"{what}: expected a device tensor")
    if t.get_device() != at:
        raise ValueError(f"{what}: on device {t.get_device()}, the current one is {at}")
    if t.dtype not in _kinds[kind]:
        raise ValueError(f"{what}: dtype {t.dtype}, expected {kind}")
    shape = t.shape
    if len(shape) == 1:
        shape = (1, shape[0])
    if len(shape) != 2 or shape[0] != n or shape[1] != dim:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, need {n} rows of {dim}")
    outer = dim
    if not t.is_contiguous():
        inner, outer = t.stride(-1), t.stride(0) if n > 1 else dim
        if dim > 1 and inner != 1 or outer < dim:
            raise ValueError(f"{what}: the values of a row must be contiguous, and rows must not overlap")
    if (n | outer) >> 31:
        raise ValueError(f"{what}: {n} rows, {outer} values apart, do not fit 32 bits")
    return t.data_ptr(), outer


def _sizes(what: str, either: int, *values):
    """The library's whole numbers are 32 bits, and ctypes cuts larger ones without
    a word.  either: the values or-ed together, which settles the usual case at once;
    negative ones are the library's to refuse."""
    if either >> 31:
        for x in values:
            if not -(1 << 31) <= x < 1 << 31:
                raise ValueError(f"{what}: {x} does not fit 32 bits")


def _ptr_tokens(t, n: int, dim: int, what: str, at: int):
    """Pointer of n rows of dim float32 values, one after the other; more rows may follow."""
    if t.numel() == n * dim and t.dtype in _kinds["f32"] and t.get_device() == at and t.is_contiguous():
        return t.data_ptr()
    p = _ptr(t, "f32", n * dim, what, at)
    if t.dim() > 1 and t.numel() != t.shape[0] * dim:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, need {n} rows of {dim}")
    return p


def _work(work, at):
    """(pointer, bytes) of a caller's workspace, or of none."""
    if work is None:
        return None, 0
    return _ptr(work, "u8", 1, "work", at), work.numel()


def _rows(t):
    return t.shape[0] if t.dim() == 2 else 1


def _stream(stream=None):
    if stream is not None:
        return C.c_void_p(stream)
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def available() -> bool:
    return bool(load().gllm_hip_available())


def stream_release(stream=None):
    """The caller will enqueue no more work on `stream` (default: torch's
    current stream): the calling thread's scratch for it is freed once it
    drains, except buffers a captured graph may still use."""
    call("gllm_hip_stream_release", _stream(stream))


class Weight:
    """A quantized GGUF tensor resident in HBM (prepareMetalWeight, model.go:2454)."""

    def __init__(self, handle, qtype, rows, cols):
        self.handle = handle
        self.type, self.rows, self.cols = qtype, rows, cols

    @classmethod
    def from_host(cls, raw, qtype: int, rows: int, cols: int) -> "Weight":
        raw = np.ascontiguousarray(raw, dtype=np.uint8)
        h = call_ptr("gllm_hip_weight_new", _np_ptr(raw), raw.nbytes, qtype, rows, cols)
        return cls(h, qtype, rows, cols)

    @classmethod
    def from_device(cls, tensor, qtype: int, rows: int, cols: int, stream=None) -> "Weight":
        h = call_ptr("gllm_hip_weight_from_device", _dev(tensor, "u8", 0, "tensor"),
                     tensor.numel() * tensor.element_size(), qtype, rows, cols, _stream(stream))
        return cls(h, qtype, rows, cols)

    def release(self):
        if self.handle:
            load().gllm_hip_weight_release(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    # host-pointer forms ----------------------------------------------------
    def matvec_into(self, x, out=None):
        x = _host_f32(x, self.cols, "matvec_into x")
        if out is None:
            out = np.empty(self.rows, np.float32)
        elif out.dtype != np.float32 or not out.flags.c_contiguous or out.size < self.rows:
            raise ValueError("matvec_into out: need a contiguous float32 array of rows elements")
        call("gllm_hip_matvec", self.handle, _np_ptr(x), _np_ptr(out))
        return out

    def matvec_batch(self, xs):
        xs = np.ascontiguousarray(xs, dtype=np.float32)
        if xs.size % self.cols:
            raise ValueError("matvec_batch: xs is not a whole number of cols-wide rows")
        xs = xs.reshape(-1, self.cols)
        out = np.empty((xs.shape[0], self.rows), np.float32)
        call("gllm_hip_matvec_batch", self.handle, _np_ptr(xs), xs.shape[0], _np_ptr(out))
        return out

    def argmax_matvec(self, x, recent=None, penalty: float = 1.0) -> int:
        """Greedy token of W.x; with recent / penalty, after applyRepeatPenalty
        (sampling.go:136-153), as ArgmaxQ6KPenalized (internal/metal/
        metal_darwin.go:1175) takes them."""
        x = _host_f32(x, self.cols, "argmax_matvec x")
        tok = C.c_uint32(0)
        if recent is None and penalty == 1.0:
            call("gllm_hip_argmax", self.handle, _np_ptr(x), C.byref(tok))
        else:
            rec = np.ascontiguousarray(recent if recent is not None else [], dtype=np.uint32)
            call("gllm_hip_argmax_penalized", self.handle, _np_ptr(x),
                 _np_ptr(rec) if rec.size else None, rec.size, float(penalty), C.byref(tok))
        return int(tok.value)

    # device forms ------------------------------------------------------------
    def matvec_dev(self, xs, out, stream=None):
        """xs: (p, cols) float32 device tensor; out: (p, >= rows) float32."""
        p = _rows(xs)
        stride = out.shape[-1]
        if xs.shape[-1] != self.cols or stride < self.rows:
            raise ValueError(f"matvec_dev: xs (.., {xs.shape[-1]}) / out (.., {stride}) do not fit "
                             f"{self.rows}x{self.cols}")
        call("gllm_hip_matvec_dev", self.handle, _dev(xs, "f32", p * self.cols, "xs"), p,
             _dev(out, "f32", p * stride, "out"), stride, _stream(stream))
        return out

    def matvec_q8_dev(self, act, p, out, stream=None):
        """Row kernels only, against activations quantised by q8k_prepare_dev."""
        stride = out.shape[-1]
        if stride < self.rows:
            raise ValueError("matvec_q8_dev: out rows shorter than the weight's rows")
        call("gllm_hip_matvec_q8_dev", self.handle, _dev(act, "u8", act_bytes(self.cols, p), "act"),
             p, _dev(out, "f32", p * stride, "out"), stride, _stream(stream))
        return out

    def argmax_dev(self, x, token_out, stream=None, recent=None, penalty: float = 1.0):
        """recent: uint32/int32 device tensor of token ids, or None."""
        xp = _dev(x, "f32", self.cols, "x")
        tp = _dev(token_out, "u32", 1, "token_out")
        if recent is None and penalty == 1.0:
            call("gllm_hip_argmax_dev", self.handle, xp, tp, _stream(stream))
        else:
            n = 0 if recent is None else recent.numel()
            call("gllm_hip_argmax_penalized_dev", self.handle, xp,
                 _dev(recent, "u32", n, "recent") if n else None, n, float(penalty), tp,
                 _stream(stream))
        return token_out

    def lane_ints_dev(self, x, out, stream=None):
        call("gllm_hip_lane_ints_dev", self.handle, _dev(x, "f32", self.cols, "x"),
             _dev(out, "i32", self.rows * (self.cols // 256) * 8, "out"), _stream(stream))
        return out

    def rows_dev(self, ids, out, stream=None):
        """(Weight).RowInto (model.go:1034) for every id in the device
        tensor ids: out[i] = row ids[i] as f32 (ids must be < rows)."""
        n = ids.numel()
        call("gllm_hip_weight_rows_dev", self.handle, _dev(ids, "u32", n, "ids"), n,
             _dev(out, "f32", n * self.cols, "out"), _stream(stream))
        return out

    def download_dev(self, out, stream=None):
        call("gllm_hip_weight_download_dev", self.handle,
             _dev(out, "u8", self.rows * row_bytes(self.type, self.cols), "out"), _stream(stream))
        return out


def matvec_multi_dev(weights, xs, outs, stream=None):
    n = len(weights)
    p = _rows(xs)
    for w, o in zip(weights, outs):
        if xs.shape[-1] != w.cols or o.shape[-1] < w.rows:
            raise ValueError("matvec_multi_dev: xs / out shapes do not fit a weight")
    hs = (C.c_void_p * n)(*[w.handle for w in weights])
    ps = (C.c_void_p * n)(*[_dev(o, "f32", p * o.shape[-1], "out").value for o in outs])
    strides = (C.c_int * n)(*[o.shape[-1] for o in outs])
    call("gllm_hip_matvec_multi_dev", n, hs, _dev(xs, "f32", p * weights[0].cols, "xs"), p, ps,
         strides, _stream(stream))


def swiglu_down_dev(gate: Weight, up: Weight, down: Weight, x, out, stream=None):
    """down . siluMulF32(gate . x, up . x) for one token (ForwardBodyInto's
    FFN, model.go:2780-2800), gate/up routed as tryMatvec2Into routes them."""
    if gate.cols != up.cols or gate.rows != up.rows or down.cols != gate.rows:
        raise ValueError("swiglu_down_dev: gate / up / down shapes do not chain")
    call("gllm_hip_swiglu_down_dev", gate.handle, up.handle, down.handle,
         _dev(x, "f32", gate.cols, "x"), _dev(out, "f32", down.rows, "out"), _stream(stream))
    return out


def _matvec_into(qtype, data, x, rows, cols, out):
    w = Weight.from_host(data, qtype, rows, cols)
    try:
        return w.matvec_into(x, out)
    finally:
        w.release()


def matvec_q4k_into(data, x, rows, cols, out=None):
    return _matvec_into(TYPE_Q4_K, data, x, rows, cols, out)


def matvec_q6k_into(data, x, rows, cols, out=None):
    return _matvec_into(TYPE_Q6_K, data, x, rows, cols, out)


def matvec_q8_0_into(data, x, rows, cols, out=None):
    return _matvec_into(TYPE_Q8_0, data, x, rows, cols, out)


def matvec2_into(a: Weight, b: Weight, x):
    x = np.ascontiguousarray(x, dtype=np.float32)
    oa, ob = np.empty(a.rows, np.float32), np.empty(b.rows, np.float32)
    call("gllm_hip_matvec2", a.handle, b.handle, _np_ptr(x), _np_ptr(oa), _np_ptr(ob))
    return oa, ob


def matvec3_into(a: Weight, b: Weight, c: Weight, x):
    x = np.ascontiguousarray(x, dtype=np.float32)
    oa, ob, oc = (np.empty(w.rows, np.float32) for w in (a, b, c))
    call("gllm_hip_matvec3", a.handle, b.handle, c.handle, _np_ptr(x), _np_ptr(oa),
         _np_ptr(ob), _np_ptr(oc))
    return oa, ob, oc


def act_bytes(cols: int, p: int = 1) -> int:
    """Bytes of the quantised-activation buffer for p rows of cols."""
    return int(load().gllm_hip_act_bytes(cols, p))


def q8k_prepare_dev(xs, act, stream=None):
    """acquireQ8 + xsums for p rows of xs into the device buffer `act`."""
    p = _rows(xs)
    cols = xs.shape[-1]
    call("gllm_hip_q8k_prepare_dev", _dev(xs, "f32", p * cols, "xs"), cols, p,
         _dev(act, "u8", act_bytes(cols, p), "act"), _stream(stream))
    return act


def q8k_quantize_dev(x, q8_out, scales_out, stream=None):
    p = _rows(x)
    cols = x.shape[-1]
    call("gllm_hip_q8k_quantize_dev", _dev(x, "f32", p * cols, "x"), cols, p,
         _dev(q8_out, "u8", p * cols, "q8_out"), _dev(scales_out, "f32", p * (cols // 256), "scales"),
         _stream(stream))


def quantize_rows_dev(qtype, src, dst, stream=None):
    rows, cols = src.shape
    call("gllm_hip_quantize_rows_dev", qtype, _dev(src, "f32", rows * cols, "src"), rows, cols,
         _dev(dst, "u8", rows * row_bytes(qtype, cols), "dst"), _stream(stream))
    return dst


def fill_normal_dev(out, seed: int, std: float, stream=None):
    call("gllm_hip_fill_normal_dev", _dev(out, "f32", 0, "out"), out.numel(), seed, std,
         _stream(stream))
    return out


class Rope:
    """Rotary positions: head layout, part of the head and scaled frequencies
    (buildRopeInvFreq model.go:1728-1799), kept on the current device.

    layout: "interleaved" (pairs 2i, 2i + 1) or "half" (i, i + rot_dim / 2);
    scaling: "none", "linear" (factor), "yarn" (factor, orig_ctx, beta_fast,
    beta_slow) or "llama3" (factor, orig_ctx, low_freq_factor,
    high_freq_factor); freq_factors: rot_dim / 2 divisors of the frequencies
    (a GGUF file's rope_freqs.weight)."""

    LAYOUTS = {"interleaved": _lib.ROPE_INTERLEAVED, "half": _lib.ROPE_HALF}
    SCALINGS = {"none": _lib.ROPE_PLAIN, "linear": _lib.ROPE_LINEAR, "yarn": _lib.ROPE_YARN, "llama3": _lib.ROPE_LLAMA3}

    def __init__(self, head_dim: int, rot_dim=None, layout="interleaved", theta: float = 500000.0, scaling="none",
                 factor: float = 1.0, orig_ctx: int = 0, low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 1.0, freq_factors=None):
        self.handle = None
        cfg = self.config(head_dim, rot_dim, layout, theta, scaling, factor, orig_ctx, low_freq_factor, high_freq_factor,
                          beta_fast, beta_slow, attn_factor, freq_factors)
        self.head_dim, self.rot_dim = cfg.head_dim, cfg.rot_dim
        self.handle = call_ptr("gllm_hip_rope_new", C.byref(cfg))

    @classmethod
    def config(cls, head_dim, rot_dim=None, layout="interleaved", theta=500000.0, scaling="none", factor=1.0, orig_ctx=0,
               low_freq_factor=1.0, high_freq_factor=4.0, beta_fast=32.0, beta_slow=1.0, attn_factor=1.0,
               freq_factors=None):
        if layout not in cls.LAYOUTS or scaling not in cls.SCALINGS:
            raise ValueError(f"Rope: layout {layout!r}, scaling {scaling!r}")
        sizes = int(head_dim), int(head_dim if rot_dim is None else rot_dim), int(orig_ctx)
        _sizes("Rope", 1 << 31, *sizes)
        c = _lib.RopeConfig()
        c.head_dim, c.rot_dim, c.orig_ctx = sizes
        c.layout, c.scaling = cls.LAYOUTS[layout], cls.SCALINGS[scaling]
        c.theta, c.factor, c.attn_factor = float(theta), float(factor), float(attn_factor)
        c.low_freq_factor, c.high_freq_factor = float(low_freq_factor), float(high_freq_factor)
        c.beta_fast, c.beta_slow = float(beta_fast), float(beta_slow)
        if freq_factors is not None:
            c._kept = _host_f32(freq_factors, c.rot_dim // 2, "Rope freq_factors")
            c.freq_factors = c._kept.ctypes.data
        return c

    @classmethod
    def frequencies(cls, *args, **kwargs):
        """(inverse frequencies, amplitude) of a configuration, in 64 bits; on the host."""
        c = cls.config(*args, **kwargs)
        inv, amp = np.empty(max(0, c.rot_dim // 2), np.float64), C.c_double(0)
        call("gllm_hip_rope_frequencies", C.byref(c), _np_ptr(inv), C.byref(amp))
        return inv, amp.value

    def apply_dev(self, x, positions, out=None, stream=None):
        """Rotate x (tokens, heads * head_dim) by positions (int32), in place without out."""
        at, current = _here()
        out = x if out is None else out
        n, dim = positions.numel(), x.shape[-1]
        heads = dim // self.head_dim
        if heads * self.head_dim != dim:
            raise ValueError(f"x: rows of {dim} are not heads of {self.head_dim}")
        xp, xs = _ptr_rows(x, "f32", n, dim, "x", at)
        op, os = _ptr_rows(out, "f32", n, dim, "out", at)
        call("gllm_hip_rope_dev", self.handle, xp, xs, n, heads, _ptr(positions, "i32", n, "positions", at), op, os,
             current if stream is None else stream)
        return out

    def release(self):
        if self.handle:
            load().gllm_hip_rope_release(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


def attend_shared_bytes(n, n_heads, n_kv_heads, hd, length, most) -> int:
    """Bytes of a workspace for KVCacheF16.attend_shared_dev."""
    _sizes("attend_shared_bytes", n | n_heads | n_kv_heads | hd | length | most, n, n_heads, n_kv_heads, hd, length, most)
    return int(load().gllm_hip_attend_shared_bytes(n, n_heads, n_kv_heads, hd, length, most))


def attend_mass_bytes(n, n_heads, n_kv_heads, hd, length) -> int:
    """Bytes of a workspace for KVCacheF16.attend_mass_dev over `length` rows."""
    _sizes("attend_mass_bytes", n | n_heads | n_kv_heads | hd | length, n, n_heads, n_kv_heads, hd, length)
    return int(load().gllm_hip_attend_mass_bytes(n, n_heads, n_kv_heads, hd, length))


def keep_bytes(layers, n_kv_heads, budget) -> int:
    """Bytes of a workspace for KVCacheF16.keep_dev."""
    _sizes("keep_bytes", layers | n_kv_heads | budget, layers, n_kv_heads, budget)
    return int(load().gllm_hip_kv_keep_bytes(layers, n_kv_heads, budget))


class _DeviceRows:
    """A cache's rows for torch.as_tensor, which keeps this object (and the cache) alive."""

    def __init__(self, cache, ptr, rows, dim):
        self.cache = cache
        self.__cuda_array_interface__ = {"shape": (rows, dim), "typestr": "<f2", "data": (ptr, False), "version": 2}


class KVCacheF16:
    """HBM-resident F16 KV cache (NewKVCacheF16, model.go:1396)."""

    def __init__(self, layers, kv_dim_k, kv_dim_v, max_len, handle=None, owned=True):
        self.layers, self.kv_dim_k, self.kv_dim_v, self.max_len = layers, kv_dim_k, kv_dim_v, max_len
        self.handle = handle or call_ptr("gllm_hip_kv_new", layers, kv_dim_k, kv_dim_v, max_len)
        self.owned = owned

    def release(self):
        if self.handle and self.owned:
            load().gllm_hip_kv_release(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    def k_ptr(self, layer):
        return load().gllm_hip_kv_k_dev(self.handle, layer)

    def v_ptr(self, layer):
        return load().gllm_hip_kv_v_dev(self.handle, layer)

    def read(self, layer, pos0, n):
        """(K rows, V rows) of positions pos0..pos0+n-1 as f16 bit arrays."""
        k = np.empty((n, self.kv_dim_k), np.uint16)
        v = np.empty((n, self.kv_dim_v), np.uint16)
        call("gllm_hip_kv_read", self.handle, layer, pos0, n, _np_ptr(k), _np_ptr(v))
        return k, v

    def store_kv(self, layer, pos, k, v):
        k = _host_f32(k, self.kv_dim_k, "store_kv k")
        v = _host_f32(v, self.kv_dim_v, "store_kv v")
        call("gllm_hip_kv_store", self.handle, layer, pos, _np_ptr(k), _np_ptr(v))

    def store_kv_dev(self, layer, pos, k, v, stream=None):
        call("gllm_hip_kv_store_dev", self.handle, layer, pos, _dev(k, "f32", self.kv_dim_k, "k"),
             _dev(v, "f32", self.kv_dim_v, "v"), _stream(stream))

    def attend_head_group(self, layer, kvh, queries, q_heads, hd, vd, start, end, scale,
                          softcap=0.0):
        queries = _host_f32(queries, q_heads * hd, "attend_head_group queries")
        out = np.empty(q_heads * vd, np.float32)
        call("gllm_hip_attend_group", self.handle, layer, kvh, _np_ptr(queries), q_heads, hd, vd,
             start, end, scale, softcap, _np_ptr(out))
        return out

    def attend_dev(self, layer, q, n_heads, n_kv_heads, hd, start, end, scale, out,
                   mode=ATTN_EXACT, stream=None):
        call("gllm_hip_attend_dev", self.handle, layer, _dev(q, "f32", n_heads * hd, "q"), n_heads,
             n_kv_heads, hd, start, end, scale, mode, _dev(out, "f32", n_heads * hd, "out"),
             _stream(stream))
        return out

    def tensors(self, layer):
        """(K, V) of a layer as float16 tensors of max_len rows over the cache's own
        memory, on its device: they hold this object, and end with release() (or, for a
        decoder's cache, with the decoder)."""
        import torch
        if not 0 <= layer < self.layers:
            raise ValueError(f"tensors: layer {layer} of {self.layers}")
        if not self.handle:
            raise ValueError("tensors: the cache is released")
        # the device by its number: on any other one, the current one too, torch would make a copy
        device = f"cuda:{load().gllm_hip_kv_device(self.handle)}"
        return tuple(torch.as_tensor(_DeviceRows(self, p, self.max_len, d), device=device)
                     for p, d in ((self.k_ptr(layer), self.kv_dim_k), (self.v_ptr(layer), self.kv_dim_v)))

    def store_rope_dev(self, layer, rope: Rope, q, k, v, positions, rows, q_out=None, stream=None):
        """Rotate q (tokens, heads * hd; or None) into q_out (default: in place) and
        k (tokens, kv heads * hd) by positions, and store k and v as f16 in the
        cache's rows (int32; outside the cache: not stored; all different)."""
        at, current = _here()
        n, hd = positions.numel(), rope.head_dim
        kd, qd = k.shape[-1], 0 if q is None else q.shape[-1]
        heads, n_kv = qd // hd, kd // hd
        if kd != n_kv * hd or qd != heads * hd:
            raise ValueError(f"store_rope_dev: q or k rows are not heads of {hd}")
        _sizes("store_rope_dev", layer, layer)
        qp = op = None
        qs = os = 0
        if q is not None:
            qp, qs = _ptr_rows(q, "f32", n, qd, "q", at)
            op, os = (qp, qs) if q_out is None else _ptr_rows(q_out, "f32", n, qd, "q_out", at)
        kp, ks = _ptr_rows(k, "f32", n, kd, "k", at)
        vp, vs = _ptr_rows(v, "f32", n, kd, "v", at)
        call("gllm_hip_kv_store_rope_dev", self.handle, layer, rope.handle, qp, qs, heads, kp, ks, vp, vs, n_kv, n,
             _ptr(positions, "i32", n, "positions", at), _ptr(rows, "i32", n, "rows", at), op, os,
             current if stream is None else stream)
        return q if q_out is None else q_out

    def attend_shared_dev(self, layer, q, n_heads, n_kv_heads, hd, start, length, starts, lens, most, scale, out,
                          work=None, stream=None):
        """One token of each request: q (requests, n_heads * hd) over the shared rows
        start .. start + length - 1 and, with most > 0, its own lens[i] rows from
        starts[i] (int32 tensors; most: the length the work is split for)."""
        at, current = _here()
        n, dim = q.shape[0] if q.dim() > 1 else 1, n_heads * hd
        _sizes("attend_shared_dev", layer | n | n_heads | n_kv_heads | hd | start | length | most,
               layer, n, n_heads, n_kv_heads, hd, start, length, most)
        wp, wb = _work(work, at)
        call("gllm_hip_attend_shared_dev", self.handle, layer, _ptr_tokens(q, n, dim, "q", at), n, n_heads, n_kv_heads,
             hd, start, length, None if starts is None else _ptr(starts, "i32", n, "starts", at),
             None if lens is None else _ptr(lens, "i32", n, "lens", at), most, scale,
             _ptr_tokens(out, n, dim, "out", at), wp, wb, current if stream is None else stream)
        return out

    def attend_mass_dev(self, layer, q, n_heads, n_kv_heads, hd, start, end, scale, mass, out, work=None, stream=None):
        """The newest tokens q (tokens, n_heads * hd), the last at row `end`, causally over
        rows start .. end; each row's weight is added to mass (n_kv_heads, >= end + 1)."""
        at, current = _here()
        n, dim, stride = q.shape[0] if q.dim() > 1 else 1, n_heads * hd, mass.shape[-1]
        _sizes("attend_mass_dev", layer | n | n_heads | n_kv_heads | hd | start | end | stride,
               layer, n, n_heads, n_kv_heads, hd, start, end, stride)
        wp, wb = _work(work, at)
        call("gllm_hip_attend_mass_dev", self.handle, layer, _ptr_tokens(q, n, dim, "q", at), n, n_heads, n_kv_heads, hd,
             start, end, scale, _ptr(mass, "f32", n_kv_heads * stride, "mass", at), stride,
             _ptr_tokens(out, n, dim, "out", at), wp, wb, current if stream is None else stream)
        return out

    def keep_dev(self, dst: "KVCacheF16", n_kv_heads, hd, length, budget, mass, pos, mass_out, pos_out, now, sinks=0,
                 recent=0, start=0, dst_start=0, work=None, stream=None):
        """Copy the budget rows of most mass (positions < sinks or >= now - recent first)
        of rows start .. start + length - 1, per layer and kv head, to dst from
        dst_start on.  mass, pos (or None: the row): (layers, n_kv_heads, rows of this
        cache); mass_out, pos_out: (layers, n_kv_heads, rows of dst)."""
        at, current = _here()
        stride, out_stride = mass.shape[-1], mass_out.shape[-1]
        if pos is not None and pos.shape[-1] != stride or pos_out.shape[-1] != out_stride:
            raise ValueError("keep_dev: mass and pos rows of different lengths")
        n = self.layers * n_kv_heads
        _sizes("keep_dev", n_kv_heads | hd | start | length | dst_start | budget | sinks | recent | now | stride | out_stride,
               n_kv_heads, hd, start, length, dst_start, budget, sinks, recent, now, stride, out_stride)
        wp, wb = _work(work, at)
        call("gllm_hip_kv_keep_dev", self.handle, dst.handle, n_kv_heads, hd, start, length, dst_start, budget, sinks,
             recent, now, _ptr(mass, "f32", n * stride, "mass", at),
             None if pos is None else _ptr(pos, "i32", n * stride, "pos", at), stride,
             _ptr(mass_out, "f32", n * out_stride, "mass_out", at), _ptr(pos_out, "i32", n * out_stride, "pos_out", at),
             out_stride, wp, wb, current if stream is None else stream)

    def evict_store_dev(self, layer, n_kv_heads, hd, k, v, start, length, mass, pos, now, sinks=0, recent=0,
                        rows_out=None, stream=None):
        """Store a token's k and v (n_kv_heads * hd, rotated) per kv head in place of the
        unprotected row of least mass among start .. start + length - 1; its pos
        becomes now (an int32 device tensor of one value), its mass 0.  mass, pos:
        (n_kv_heads, rows); rows_out: n_kv_heads int32, the rows given up."""
        at, current = _here()
        stride, dim = mass.shape[-1], n_kv_heads * hd
        if pos.shape[-1] != stride:
            raise ValueError("evict_store_dev: mass and pos rows of different lengths")
        _sizes("evict_store_dev", layer | n_kv_heads | hd | start | length | sinks | recent | stride,
               layer, n_kv_heads, hd, start, length, sinks, recent, stride)
        call("gllm_hip_kv_evict_store_dev", self.handle, layer, n_kv_heads, hd, _ptr(k, "f32", dim, "k", at),
             _ptr(v, "f32", dim, "v", at), start, length, sinks, recent,
             _ptr(mass, "f32", n_kv_heads * stride, "mass", at), _ptr(pos, "i32", n_kv_heads * stride, "pos", at), stride,
             _ptr(now, "i32", 1, "now", at), None if rows_out is None else _ptr(rows_out, "i32", n_kv_heads, "rows_out", at),
             current if stream is None else stream)
