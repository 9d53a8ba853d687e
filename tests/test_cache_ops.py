"""CPU checks of the cache operators: the arithmetic that splits attention over
workgroups, rotary frequencies, and the calls that are refused (before
anything touches a device)."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

import gopherllm_amd as g
from gopherllm_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "attn_plan.h"
using namespace gllm;
static void need(bool ok, const char* what, int n, int h, int g, int len, int most) {
    if (!ok) { std::printf("%s: n %d heads %d/%d len %d most %d\n", what, n, h, g, len, most); std::exit(1); }
}
int main() {
    const int ns[] = {1, 2, 3, 7, 16, 33, 64, 257, 4096}, rs[] = {1, 2, 4, 5, 7, 8, 17, 32, 71}, gs[] = {1, 2, 5, 8, 96};
    const int lens[] = {0, 1, 31, 32, 127, 128, 129, 300, 4001, 32768, 131072, 1 << 30};
    long plans = 0;
    for (int n : ns) for (int r : rs) for (int g : gs) for (int len : lens) for (int most : lens) {
        const int h = r * g;
        if ((long long)n * h > (1 << 24)) continue;
        const SeqPlan p = seq_plan(n, h, g, r % 2 ? 128 : 40, len, most);
        plans++;
        need(p.r == r && p.rows == (size_t)n * h, "rows", n, h, g, len, most);
        need((long long)p.row_blocks * 16 * p.nq * p.rw >= (long long)n * r, "row blocks", n, h, g, len, most);
        need(p.chunks <= kSeqMaxSplits && p.splits <= kSeqMaxSplits && p.slots == p.chunks + p.splits, "slots", n, h, g, len, most);
        need((len > 0) == (p.chunks > 0) && (most > 0) == (p.splits > 0), "parts", n, h, g, len, most);
        if (len) {
            need(p.chunk % kSeqQuantum == 0, "chunk", n, h, g, len, most);
            need((long long)p.chunk * p.chunks >= len && (long long)p.chunk * (p.chunks - 1) < len, "cover", n, h, g, len, most);
        }
        if (most) need(p.own_blocks * 16 >= r, "own blocks", n, h, g, len, most);
        need(seq_floats(p, 128) >= p.rows * (size_t)p.slots * 130, "floats", n, h, g, len, most);
        if (len && !most)
            for (int hd : {8, 40, 96, 128}) {
                const MassSpace m = mass_space(p, hd, g, len);
                const int kk = hd <= 32 ? 1 : hd <= 64 ? 2 : hd <= 96 ? 3 : 4;
                need(m.kept == (n == 1 && r <= 16), "kept", n, h, g, len, hd);
                need(m.parts % 4 == 0 && m.scale % 4 == 0 && m.ml % 4 == 0, "aligned", n, h, g, len, hd);
                if (m.kept) need(m.sstride >= len && m.sstride % 4 == 0 && m.parts == p.rows * (size_t)m.sstride, "scores", n, h, g, len, hd);
                else need(16LL * m.tiles >= (long long)n * r && m.scale == (size_t)g * m.tiles * 2 * kk * 64 * 4 &&
                          m.ml >= m.scale + (size_t)g * m.tiles * 16 && m.parts >= m.ml + 2 * p.rows, "operands", n, h, g, len, hd);
                need(mass_floats(p, hd, g, len) >= m.parts + p.rows * (size_t)p.slots * (2 + hd), "mass floats", n, h, g, len, hd);
            }
    }
    const int big = 2147483647;
    struct { int s, l, m, a, b; } cut[] = {{0, 5, 10, 0, 5}, {7, 5, 10, 7, 10}, {-3, 5, 10, 0, 2}, {-9, 5, 10, 0, 0}, {12, 5, 10, 10, 10},
        {3, 0, 10, 3, 3}, {3, -4, 10, 3, 3}, {big, big, 10, 10, 10}, {-big, big, 10, 0, 0}, {5, big, 10, 5, 10}, {-5, big, big, 0, big - 5}};
    for (auto& c : cut) {
        const RowSpan s = clip_rows(c.s, c.l, c.m);
        need(s.a == c.a && s.b == c.b, "clip", c.s, c.l, c.m, s.a, s.b);
    }
    std::printf("%ld plans\n", plans);
}
"""


def test_the_plan_covers_every_row(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "gopherllm_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


# --- rotary frequencies -------------------------------------------------------


def test_plain_and_linear_frequencies():
    inv, amp = g.Rope.frequencies(128, 96, theta=10000.0, attn_factor=1.5)
    want = 10000.0 ** (-np.arange(48) / 48.0)
    assert np.allclose(inv, want, rtol=1e-15, atol=0) and amp == 1.5
    inv4, _ = g.Rope.frequencies(128, 96, theta=10000.0, scaling="linear", factor=4.0)
    assert np.allclose(inv4, want / 4, rtol=1e-15, atol=0)
    f = np.linspace(1, 8, 48).astype(np.float32)
    invf, _ = g.Rope.frequencies(128, 96, theta=10000.0, freq_factors=f)
    assert np.allclose(invf, want / f, rtol=1e-15, atol=0)


def test_llama3_frequencies():
    """Short waves stay, long ones are divided, and the two meet at the edges."""
    inv, _ = g.Rope.frequencies(128, scaling="llama3", factor=8.0, orig_ctx=8192)
    raw = 500000.0 ** (-np.arange(64) / 64.0)
    turns = 8192 * raw / (2 * np.pi)
    assert np.allclose(inv[turns >= 4], raw[turns >= 4], rtol=1e-14) and np.allclose(inv[turns <= 1], raw[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert mid.any()
    t = (turns[mid] - 1) / 3
    assert np.allclose(inv[mid], (1 - t) * raw[mid] / 8 + t * raw[mid], rtol=1e-14)


def test_yarn_frequencies():
    inv, amp = g.Rope.frequencies(128, theta=10000.0, scaling="yarn", factor=16.0, orig_ctx=4096)
    raw = 10000.0 ** (-np.arange(64) / 64.0)
    assert amp == pytest.approx(0.1 * math.log(16.0) + 1.0, rel=1e-15)
    lo = math.floor(128 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    assert 0 < lo < hi < 64
    assert np.allclose(inv[:lo + 1], raw[:lo + 1], rtol=1e-14) and np.allclose(inv[hi:], raw[hi:] / 16, rtol=1e-14)
    assert (np.diff(inv) < 0).all()


@pytest.mark.parametrize("kw", [
    dict(head_dim=0), dict(head_dim=2000), dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=130), dict(theta=1.0),
    dict(theta=float("nan")), dict(theta=-5.0), dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=float("inf")),
    dict(scaling="yarn", factor=2.0), dict(scaling="yarn", factor=2.0, orig_ctx=100, beta_fast=1.0, beta_slow=2.0),
    dict(scaling="llama3", factor=2.0, orig_ctx=100, low_freq_factor=4.0, high_freq_factor=4.0), dict(attn_factor=0.0),
    dict(freq_factors=np.zeros(64, np.float32)), dict(freq_factors=np.full(64, 1e-20, np.float32)), dict(freq_factors=np.full(64, np.nan, np.float32))])
def test_rope_refusals(kw):
    args = dict(head_dim=128)
    args.update(kw)
    for make in (g.Rope.frequencies, g.Rope):
        with pytest.raises(g.GllmError):
            make(**args)


def test_rope_names():
    for kw in (dict(layout="pairs"), dict(scaling="ntk"), dict(freq_factors=np.ones(3, np.float32))):
        with pytest.raises(ValueError):
            g.Rope.frequencies(128, **kw)


# --- refusals -----------------------------------------------------------------


class Cache(C.Structure):
    """csrc/kv_cache.h, for caches that only a refusing call looks at."""
    _fields_ = [(n, C.c_int) for n in ("layers", "kv_dim_k", "kv_dim_v", "max_len")] + [
        ("k", C.c_void_p), ("v", C.c_void_p), ("device", C.c_int)]


def cache(layers=2, kd=256, vd=256, rows=100):
    return Cache(layers, kd, vd, rows, 0, 0, 0)


P = C.c_void_p(4096)  # an aligned address that is never read


def refused(name, code, *args):
    rc = getattr(g.load(), name)(*args)
    assert rc == code, (name, rc, _lib.last_error())
    assert _lib.last_error()


SHARED = dict(kv=None, l=0, q=P, n=3, heads=8, kvh=2, hd=64, start=0, len=10, starts=P, lens=P, most=4, scale=0.1, out=P,
              work=None, wb=0, stream=None)
MASS = dict(kv=None, l=0, q=P, n=3, heads=8, kvh=2, hd=64, start=0, end=9, scale=0.1, mass=P, stride=100, out=P, work=None,
            wb=0, stream=None)
ATTEND = [dict(n=0), dict(n=-1), dict(heads=7), dict(kvh=0), dict(heads=0), dict(hd=0), dict(hd=12), dict(hd=136), dict(q=None),
          dict(out=None), dict(l=2), dict(l=-1), dict(kvh=8, heads=8), dict(kv=None), dict(q=C.c_void_p(4100)),
          dict(out=C.c_void_p(4104)), dict(n=1 << 22)]


@pytest.mark.parametrize("kw", ATTEND + [dict(start=-1), dict(len=-1), dict(start=95), dict(start=2**31 - 1), dict(most=-1),
                                         dict(most=0), dict(starts=None), dict(lens=None)])
def test_attend_shared_refusals(kw):
    kv = cache()
    args = dict(SHARED, kv=C.byref(kv))
    args.update(kw)
    refused("gllm_hip_attend_shared_dev", g.EINVAL, *args.values())


@pytest.mark.parametrize("kw", ATTEND + [dict(start=-1), dict(end=100), dict(end=1), dict(start=8), dict(end=-1), dict(mass=None),
                                         dict(stride=9)])
def test_attend_mass_refusals(kw):
    kv = cache()
    args = dict(MASS, kv=C.byref(kv))
    args.update(kw)
    refused("gllm_hip_attend_mass_dev", g.EINVAL, *args.values())


def test_attend_needs_aligned_rows_and_32_bit_rows():
    for kv in (cache(kd=260), cache(vd=257), cache(rows=(1 << 30) + 1), cache(kd=(1 << 24) + 8)):
        refused("gllm_hip_attend_shared_dev", g.EUNSUP, *dict(SHARED, kv=C.byref(kv)).values())
        refused("gllm_hip_attend_mass_dev", g.EUNSUP, *dict(MASS, kv=C.byref(kv)).values())


def test_workspace_sizes():
    assert g.attend_shared_bytes(0, 8, 2, 64, 1, 0) == 0 and g.attend_shared_bytes(1, 8, 3, 64, 1, 0) == 0
    assert g.attend_shared_bytes(4, 8, 2, 64, 100, 9) > 0 and g.attend_mass_bytes(4, 8, 2, 64, 100) > 4 * 8 * 100 * 4 and g.attend_mass_bytes(1, 8, 2, 129, 100) == 0
    assert g.attend_mass_bytes(1, 8, 2, 64, 0) == 0
    assert g.keep_bytes(3, 2, 5) == 120 and g.keep_bytes(0, 2, 5) == 0


KEEP = dict(src=None, dst=None, kvh=2, hd=64, start=0, len=50, dst_start=0, budget=20, sinks=1, recent=2, now=50, mass=P, pos=P,
            stride=100, mass_out=C.c_void_p(1 << 20), pos_out=C.c_void_p(1 << 21), out_stride=30, work=None, wb=0, stream=None)


@pytest.mark.parametrize("kw", [
    dict(kvh=0), dict(hd=0), dict(hd=12), dict(len=0), dict(budget=0), dict(budget=51), dict(sinks=-1), dict(recent=-1), dict(now=-1),
    dict(src=None), dict(dst=None), dict(mass=None), dict(mass_out=None), dict(pos_out=None), dict(kvh=8), dict(start=60), dict(start=-1),
    dict(dst_start=-1), dict(dst_start=15), dict(stride=49), dict(out_stride=19), dict(mass_out=P), dict(pos_out=C.c_void_p(4096 + 800))])
def test_keep_refusals(kw):
    src, dst = cache(), cache(rows=30)
    args = dict(KEEP, src=C.byref(src), dst=C.byref(dst))
    args.update(kw)
    refused("gllm_hip_kv_keep_dev", g.EINVAL, *args.values())


def test_keep_refuses_itself_other_layers_and_unaligned_rows():
    a, b = cache(), cache(layers=3)
    refused("gllm_hip_kv_keep_dev", g.EINVAL, *dict(KEEP, src=C.byref(a), dst=C.byref(a)).values())
    refused("gllm_hip_kv_keep_dev", g.EINVAL, *dict(KEEP, src=C.byref(a), dst=C.byref(b)).values())
    c = cache(kd=260)
    refused("gllm_hip_kv_keep_dev", g.EUNSUP, *dict(KEEP, src=C.byref(a), dst=C.byref(c)).values())
    big, to = cache(kd=1 << 20, vd=1 << 20, rows=1 << 20), cache(kd=1 << 20, vd=1 << 20, rows=1 << 20)
    refused("gllm_hip_kv_keep_dev", g.EUNSUP, *dict(KEEP, src=C.byref(big), dst=C.byref(to), kvh=1 << 14, len=1 << 20, budget=1 << 20,
                                                    stride=1 << 20, out_stride=1 << 20).values())
    far = cache(rows=(1 << 30) + 1)
    refused("gllm_hip_kv_keep_dev", g.EUNSUP, *dict(KEEP, src=C.byref(far), dst=C.byref(a)).values())
    refused("gllm_hip_kv_evict_store_dev", g.EUNSUP, *dict(EVICT, kv=C.byref(far)).values())


EVICT = dict(kv=None, l=0, kvh=2, hd=64, k=P, v=P, start=0, len=50, sinks=1, recent=2, mass=P, pos=P, stride=100, now=P, rows=None,
             stream=None)


@pytest.mark.parametrize("kw", [
    dict(kvh=0), dict(hd=0), dict(hd=2000), dict(len=0), dict(sinks=-1), dict(recent=-1), dict(k=None), dict(v=None), dict(mass=None),
    dict(pos=None), dict(now=None), dict(l=2), dict(kvh=5), dict(start=51), dict(start=-1), dict(stride=49), dict(kv=None)])
def test_evict_refusals(kw):
    kv = cache()
    args = dict(EVICT, kv=C.byref(kv))
    args.update(kw)
    refused("gllm_hip_kv_evict_store_dev", g.EINVAL, *args.values())


def test_rope_calls_without_a_rope():
    refused("gllm_hip_rope_dev", g.EINVAL, None, P, 64, 1, 1, P, P, 64, None)
    kv = cache()
    refused("gllm_hip_kv_store_rope_dev", g.EINVAL, C.byref(kv), 0, None, P, 64, 1, P, 64, P, 64, 1, 1, P, P, P, 64, None)
