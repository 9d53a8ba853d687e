"""CPU checks of the calls for drafted tokens and for copied rows: how the work is
split, in which order rows are copied, what is refused (before anything touches a
device) and what the Python side passes on."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import gopherllm_amd as g
from gopherllm_amd import _lib, api
from test_cache_calls import FAR, Tensor, calls, fresh, ints  # noqa: F401
from test_cache_calls import cache as py_cache
from test_cache_ops import P, cache, refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, program):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "gopherllm_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "attn_plan.h"
using namespace gllm;
static void need(bool ok, const char* what, int n, int m, int h, int g, int hd, int most) {
    if (!ok) { std::printf("%s: n %d m %d heads %d/%d of %d most %d\n", what, n, m, h, g, hd, most); std::exit(1); }
}
int main() {
    const int ns[] = {1, 2, 3, 7, 16, 33, 64, 257}, ms[] = {1, 2, 3, 4, 5, 8, 13, 16, 17, 31, 33, 64, 65, 128, 129, 255, 256};
    const int rs[] = {1, 2, 4, 5, 7, 8, 17, 32}, gs[] = {1, 2, 5, 8, 96}, hds[] = {8, 40, 64, 96, 128};
    const int mosts[] = {0, 1, 31, 127, 128, 129, 300, 2000, 4001, 8192, 8193, 32768, 131072, 1 << 30, 2147483647};
    for (int g : gs) for (int r : rs) for (int hd : hds) {
        size_t smaller[257] = {};
        for (int n : ns) {
            size_t before_m = 0;
            for (int m : ms) {
                const int h = r * g;
                if ((long long)n * m * h > (1 << 22)) continue;
                size_t before = 0;
                for (int most : mosts) {
                    const TreePlan p = tree_plan(n, m, h, g, hd, most);
                    need(p.r == r && p.rows == (size_t)n * m * h, "rows", n, m, h, g, hd, most);
                    need(16LL * p.nq * p.rw * p.row_blocks >= (long long)m * r, "row blocks", n, m, h, g, hd, most);
                    need(16LL * p.nq * p.rw * (p.row_blocks - 1) < (long long)m * r, "empty block", n, m, h, g, hd, most);
                    need(p.splits >= 1 && p.splits <= kSeqMaxSplits, "splits", n, m, h, g, hd, most);
                    need(p.target >= 1 && p.units >= 1 && p.units <= p.target + (long long)n * p.row_blocks, "units", n, m, h, g, hd, most);
                    need((long long)g * p.units < (1 << 23), "launch", n, m, h, g, hd, most);
                    need(p.parts >= p.rows * (size_t)p.splits, "room", n, m, h, g, hd, most);
                    // any lengths make no more units and parts than that, each request at least one for a block
                    for (int seed = 0; seed < 4; seed++) {
                        long long total = 0, longest = 0, units = 0;
                        const auto len = [&](int i) { return (long long)(((i * 2654435761u + seed * 40503u) >> 7) % (seed ? seed * 5000 : 1) + m) * (seed == 3 && i ? 0 : 1) + 1; };
                        for (int i = 0; i < n; i++) total += len(i) * p.row_blocks, longest = std::max(longest, len(i));
                        long long chunk = std::max((total + p.target - 1) / p.target, (longest + p.splits - 1) / p.splits);
                        chunk = (chunk + kSeqQuantum - 1) / kSeqQuantum * kSeqQuantum;
                        for (int i = 0; i < n; i++) {
                            need((len(i) + chunk - 1) / chunk <= p.splits, "parts of a range", n, m, h, g, hd, most);
                            units += (len(i) + chunk - 1) / chunk * p.row_blocks;
                        }
                        need(units <= p.units, "units made", n, m, h, g, hd, most);
                    }
                    const size_t f = tree_floats(p, n, hd);
                    need(f >= before, "never falls as contexts grow", n, m, h, g, hd, most);
                    before = f;
                }
                need(before >= before_m, "never falls as trees grow", n, m, h, g, hd, 1 << 30);
                need(before >= smaller[m], "never falls as requests grow", n, m, h, g, hd, 1 << 30);
                before_m = smaller[m] = before;
            }
        }
    }
}
"""


def test_the_tree_plan_covers_every_row_and_its_room_never_falls(tmp_path):
    run(tmp_path, PLAN)


MANY_KV_HEADS = r"""
#include <cstdio>
#include "attn_plan.h"
using namespace gllm;
int main() {
    const int gs[] = {255, 256, 257, 511, 512, 513, 514, 534, 600, 1023, 1024, 1025, 4096}, rs[] = {1, 2, 3, 16, 32}, ns[] = {1, 2, 3, 4, 5, 8, 1000};
    const int ms[] = {1, 4, 15, 16, 17, 64, 65, 256}, mosts[] = {0, 128, 300, 497, 1000, 4001, 32768, 1 << 30, 2147483647};
    for (int hd : {8, 64, 128}) for (int g : gs) for (int r : rs) for (int n : ns) for (int m : ms) {
        if ((long long)n * m * r * g > (1 << 22) || (long long)m * r > (1 << 20)) continue;
        size_t before = 0;
        for (int most : mosts) {
            const TreePlan p = tree_plan(n, m, r * g, g, hd, most);
            // the outputs, bases and sums of all parts, and each request's number of parts behind them
            const size_t end = p.rows * (size_t)p.splits * (hd + 2) + n, room = tree_floats(p, n, hd);
            if (p.rows * (size_t)p.splits > p.parts || end > room || room < before || p.splits < 1 || p.splits > kSeqMaxSplits ||
                p.units > (long long)n * p.row_blocks * p.splits || (long long)g * p.units >= 1 << 23)
                return std::printf("n %d m %d heads %d/%d of %d most %d: %zu rows of %d parts, room for %zu\n", n, m, r * g, g, hd, most, p.rows, p.splits, p.parts), 1;
            before = room;
        }
    }
}
"""


def test_parts_fit_their_room_for_any_number_of_kv_heads(tmp_path):
    """A workgroup for each kv head is more than are wanted from 512 kv heads on."""
    run(tmp_path, MANY_KV_HEADS)


COPY = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "copy_plan.h"
using namespace gllm;
int main() {
    std::mt19937 rng(5);
    const auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long ways[3] = {0, 0, 0}, refused = 0;
    for (int trial = 0; trial < 20000; trial++) {
        const int rows = pick(1, 60), n = pick(0, 7), kind = trial % 4;
        std::vector<int32_t> m;
        int at = 0, to = 0;
        for (int i = 0; i < n; i++) {
            int len = pick(0, 9), src, dst;
            if (kind == 0) src = pick(0, rows), dst = pick(0, rows);                     // anything
            else if (kind == 1) at += pick(0, 5), src = at, dst = to, at += len, to += len;  // down over gaps
            else if (kind == 2) src = pick(0, rows), dst = to, to += len + pick(0, 2);    // destinations apart
            else src = pick(0, 5) * 9, dst = i * 9, len = 9;                              // exchanged places
            if (src + len > rows || dst + len > rows) continue;
            m.insert(m.end(), {src, dst, len});
        }
        const int k = (int)m.size() / 3;
        std::vector<int> written(rows, 0), want(rows), got(rows);
        bool apart = true;
        for (int r = 0; r < rows; r++) want[r] = got[r] = r;
        for (int i = 0; i < k; i++)
            for (int r = 0; r < m[3 * i + 2]; r++) {
                apart &= !written[m[3 * i + 1] + r]++;
                want[m[3 * i + 1] + r] = m[3 * i] + r;
            }
        const CopyPlan p = copy_plan(m.data(), k, true), other = copy_plan(m.data(), k, false);
        if (p.ok != apart || other.ok != apart || (apart && (!other.apart || !other.staged.empty()))) return std::printf("trial %d: ok\n", trial), 1;
        if (!apart) { refused++; continue; }
        ways[p.apart ? 0 : p.staged.empty() ? 1 : 2]++;
        const size_t c = p.moves.size();
        std::vector<int> aside;
        for (const RowMove& x : p.staged)
            for (int r = 0; r < x.rows; r++) aside.push_back(got[x.src + r]);
        if (p.apart) {  // in any order, row by row
            for (size_t i = c; i-- > 0;)
                for (int r = 0; r < p.moves[i].rows; r++) got[p.moves[i].dst + r] = got[p.moves[i].src + r];
        } else {  // `tile` rows read, then written; a move over its own rows from the right end
            const int tile = pick(1, 12);
            std::vector<int> from, into;
            for (const RowMove& x : p.moves)
                for (int r = 0; r < x.rows; r++) {
                    const int o = x.dst < x.src ? r : x.rows - 1 - r;
                    from.push_back(x.src + o);
                    into.push_back(x.dst + o);
                }
            for (size_t r0 = 0; r0 < from.size(); r0 += tile) {
                std::vector<int> held;
                const size_t end = std::min(from.size(), r0 + tile);
                for (size_t r = r0; r < end; r++) held.push_back(got[from[r]]);
                for (size_t r = end; r-- > r0;) got[into[r]] = held[r - r0];
            }
        }
        size_t o = 0;
        for (const RowMove& x : p.staged)
            for (int r = 0; r < x.rows; r++) got[x.dst + r] = aside[o++];
        if (p.apart && o) return std::printf("trial %d: set aside for nothing\n", trial), 1;
        if (got != want) return std::printf("trial %d: apart %d, %zu set aside\n", trial, (int)p.apart, p.staged.size()), 1;
    }
    if (ways[0] < 500 || ways[1] < 500 || ways[2] < 200 || refused < 500) return std::printf("%ld %ld %ld %ld\n", ways[0], ways[1], ways[2], refused), 1;
}
"""


def test_rows_are_read_before_they_are_written(tmp_path):
    run(tmp_path, COPY)


CIRCLES = r"""
#include <cstdio>
#include <random>
#include "copy_plan.h"
using namespace gllm;
// Whether move x is on a circle of moves, each of which writes rows that the next reads
static bool on_circle(const std::vector<RowMove>& all, const RowMove& x) {
    const auto before = [](const RowMove& a, const RowMove& b) { return a.src < b.dst + b.rows && b.dst < a.src + a.rows; };
    std::vector<char> seen(all.size(), 0);
    std::vector<RowMove> now{x};
    while (!now.empty()) {
        const RowMove a = now.back();
        now.pop_back();
        for (size_t i = 0; i < all.size(); i++) {
            if (all[i].dst == a.dst || !before(a, all[i])) continue;  // destinations tell moves apart
            if (all[i].dst == x.dst) return true;
            if (!seen[i]++) now.push_back(all[i]);
        }
    }
    return false;
}
static long rows_of(const std::vector<RowMove>& v) {
    long n = 0;
    for (const RowMove& x : v) n += x.rows;
    return n;
}
int main() {
    // places 0 and 1 of 1000 rows exchanged, and moves of fewer rows that wait for them and for each other
    for (int waiting : {0, 1, 2, 18, 300})
        for (int less : {1, 499, 999}) {
            std::vector<int32_t> m{0, 1000, 1000, 1000, 0, 1000};
            for (int i = 0; i < waiting; i++) m.insert(m.end(), {1000 * (i + 2), i ? 1000 * (i + 1) : 500, less < 500 || i ? less : 500});
            if (waiting) m[5] = 500;  // the first of them goes to rows that the exchange reads
            const CopyPlan p = copy_plan(m.data(), (int)m.size() / 3, true);
            const long least = waiting ? 500 : 1000;
            if (!p.ok || p.staged.size() != 1 || rows_of(p.staged) != least) return std::printf("%d waiting: %zu moves of %ld rows set aside, not %ld\n", waiting, p.staged.size(), rows_of(p.staged), least), 1;
        }
    // any moves of places, some of several to one source
    std::mt19937 rng(7);
    long circles = 0, none = 0;
    for (int trial = 0; trial < 3000; trial++) {
        const int n = 2 + (int)(rng() % 30);
        std::vector<int32_t> m;
        for (int i = 0; i < n; i++) {
            const int rows = 1 + (int)(rng() % 9), at = (int)(rng() % (unsigned)n);
            m.insert(m.end(), {10 * at + (int)(rng() % (unsigned)(10 - rows + 1)), 10 * i, rows});
        }
        const CopyPlan p = copy_plan(m.data(), n, true);
        std::vector<RowMove> all = p.moves;
        all.insert(all.end(), p.staged.begin(), p.staged.end());
        bool any = false;
        for (const RowMove& x : all) any |= on_circle(all, x);
        for (const RowMove& x : p.staged)
            if (!on_circle(all, x)) return std::printf("trial %d: rows %d of %d moves set aside, in no circle\n", trial, x.rows, n), 1;
        if (any == p.staged.empty()) return std::printf("trial %d: circles %d, %zu set aside\n", trial, (int)any, p.staged.size()), 1;
        (any ? circles : none)++;
    }
    if (circles < 300 || none < 300) return std::printf("%ld %ld\n", circles, none), 1;
    // as many moves as a call takes: one circle of all, and circles of two
    std::vector<int32_t> ring, pairs;
    for (int i = 0; i < kCopyMost; i++) {
        ring.insert(ring.end(), {4 * i, 4 * ((i + 1) % kCopyMost), i == 77 ? 3 : 4});
        pairs.insert(pairs.end(), {4 * i, 4 * (i ^ 1), 4});
    }
    const CopyPlan p = copy_plan(ring.data(), kCopyMost, true), q = copy_plan(pairs.data(), kCopyMost, true);
    if (rows_of(p.staged) != 3 || q.staged.size() != kCopyMost / 2) return std::printf("%ld rows, %zu moves\n", rows_of(p.staged), q.staged.size()), 1;
}
"""


def test_only_rows_of_a_circle_are_set_aside(tmp_path):
    run(tmp_path, CIRCLES)


# --- refusals -----------------------------------------------------------------

TREE = dict(kv=None, l=0, q=P, n=3, m=4, heads=8, kvh=2, hd=64, starts=P, lens=P, most=10, parents=P, counts=P, scale=0.1, out=P,
            work=None, wb=0, stream=None)


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=-1), dict(n=2**31 - 1), dict(m=0), dict(m=-3), dict(m=257), dict(heads=7), dict(kvh=0), dict(heads=0), dict(hd=0),
    dict(hd=12), dict(hd=136), dict(q=None), dict(out=None), dict(starts=None), dict(lens=None), dict(parents=None), dict(l=2), dict(l=-1),
    dict(kvh=8, heads=8), dict(kv=None), dict(q=C.c_void_p(4100)), dict(out=C.c_void_p(4104)), dict(n=1 << 18, m=4), dict(most=-1)])
def test_attend_tree_refusals(kw):
    kv = cache()
    refused("gllm_hip_attend_tree_dev", g.EINVAL, *{**TREE, "kv": C.byref(kv), **kw}.values())


def test_attend_tree_needs_aligned_rows_and_32_bit_rows():
    for kv in (cache(kd=260), cache(vd=257), cache(rows=(1 << 30) + 1), cache(kd=(1 << 24) + 8)):
        refused("gllm_hip_attend_tree_dev", g.EUNSUP, *{**TREE, "kv": C.byref(kv)}.values())


ACCEPT = dict(logits=P, stride=100, vocab=100, n=3, m=4, tokens=P, parents=P, counts=P, temperature=0.0, uniforms=None, path=P,
              accepted=P, next=P, work=None, wb=0, stream=None)


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(n=-1), dict(m=0), dict(m=257), dict(vocab=0), dict(stride=99), dict(vocab=-5), dict(logits=None), dict(tokens=None),
    dict(parents=None), dict(path=None), dict(accepted=None), dict(next=None), dict(temperature=0.5), dict(uniforms=P),
    dict(temperature=-1.0, uniforms=P), dict(temperature=float("nan"), uniforms=P), dict(temperature=float("inf"), uniforms=P),
    dict(temperature=1e-12, uniforms=P), dict(n=1 << 24), dict(vocab=(1 << 30) + 1, stride=(1 << 30) + 1), dict(n=2**31 - 1, m=256),
    dict(work=P, wb=8), dict(work=C.c_void_p(4100), wb=1 << 30)])
def test_accept_tree_refusals(kw):
    refused("gllm_hip_accept_tree_dev", g.EINVAL, *{**ACCEPT, **kw}.values())


PATH = dict(kv=None, n=3, m=4, starts=P, lens=P, path=P, accepted=P, stream=None)


@pytest.mark.parametrize("kw", [dict(n=0), dict(n=-1), dict(n=65536), dict(m=0), dict(kv=None), dict(starts=None), dict(lens=None), dict(path=None),
                                dict(accepted=None)])
def test_keep_path_refusals(kw):
    kv = cache()
    refused("gllm_hip_kv_keep_path_dev", g.EINVAL, *{**PATH, "kv": C.byref(kv), **kw}.values())


def moves(*rows):
    return np.array(rows, np.int32).reshape(-1, 3)


@pytest.mark.parametrize("m", [
    moves((0, 5, -1)), moves((-1, 5, 2)), moves((0, -5, 2)), moves((99, 0, 2)), moves((0, 99, 2)), moves((2**31 - 1, 0, 1)), moves((0, 2**31 - 1, 1)),
    moves((5, 5, 2**31 - 1)), moves((0, 10, 5), (20, 14, 5)), moves((0, 10, 5), (10, 10, 5)), moves((0, 10, 1), (1, 10, 1))])
def test_copy_refusals(m):
    a, b = cache(), cache()
    for to in (a, b):
        refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, C.byref(a), C.byref(to), m.ctypes.data_as(C.c_void_p), len(m), None, 0, None)
        assert g.load().gllm_hip_kv_copy_rows_bytes(C.byref(a), C.byref(to), m.ctypes.data_as(C.c_void_p), len(m)) == 0


def test_copy_refuses_other_caches_and_too_many_moves():
    a, m = cache(), np.zeros((4097, 3), np.int32)
    p = m.ctypes.data_as(C.c_void_p)
    for other in (cache(layers=3), cache(kd=128), cache(vd=128)):
        refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, C.byref(a), C.byref(other), p, 1, None, 0, None)
    for n in (-1, 4097):
        refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, C.byref(a), C.byref(a), p, n, None, 0, None)
    refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, C.byref(a), C.byref(a), None, 1, None, 0, None)
    refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, None, C.byref(a), p, 1, None, 0, None)
    refused("gllm_hip_kv_copy_rows_dev", g.EINVAL, C.byref(a), None, p, 1, None, 0, None)


def test_workspace_sizes():
    for wrong in ((0, 4, 8, 2, 64, 9), (1, 0, 8, 2, 64, 9), (1, 257, 8, 2, 64, 9), (1, 4, 8, 3, 64, 9), (1, 4, 8, 2, 60, 9), (1, 4, 8, 2, 136, 9),
                  (1, 4, 8, 2, 64, -1), (1 << 18, 4, 8, 2, 64, 9)):
        assert g.attend_tree_bytes(*wrong) == 0
    assert g.attend_tree_bytes(2, 4, 8, 2, 64, 2**31 - 1) >= g.attend_tree_bytes(2, 4, 8, 2, 64, 1 << 30) > 0  # longer than any cache
    assert g.attend_tree_bytes(2, 4, 8, 2, 64, 1000) > 2 * 4 * 8 * 66 * 4
    assert g.accept_tree_bytes(2, 3, 100) >= 2 * 3 * 16 and g.accept_tree_bytes(1, 257, 100) == 0 and g.accept_tree_bytes(0, 3, 100) == 0
    assert g.accept_tree_bytes(1, 3, 0) == 0 and g.accept_tree_bytes(1 << 24, 1, 100) == 0

    def staged(m, **kw):
        a = cache(rows=9000, **kw)
        return g.load().gllm_hip_kv_copy_rows_bytes(C.byref(a), C.byref(a), m.ctypes.data_as(C.c_void_p), len(m))
    row = (1024 + 1536) * 2 * 8
    many = dict(layers=8, kd=1024, vd=1536)
    assert staged(moves((0, 1000, 1000), (1000, 0, 1000)), **many) == 1000 * row  # one of the two is set aside
    assert staged(moves((0, 1000, 1000), (1000, 2000, 1000)), **many) == 0 and staged(moves((5, 0, 5000)), **many) == 0
    assert staged(moves((0, 10, 10), (10, 0, 10)), **many) == 0  # all read at once
    few = dict(layers=1, kd=64, vd=64)
    assert staged(moves((0, 3000, 3000), (3000, 6000, 3000)), **few) == 6000 * 256  # too few workgroups to go in order
    assert staged(moves((0, 1000, 1000), (1000, 2000, 1000)), **few) == 0 and staged(moves((0, 5000, 1000)), **few) == 0 and staged(moves((5, 0, 500)), **few) == 0


def test_what_goes_in_order_is_decided_by_the_layers_of_a_launch():
    """Workgroups own 128 bytes of a layer's rows: fewer than 96 of them in a launch read many rows twice."""
    def staged(m, rows, **kw):
        a = cache(rows=rows, **kw)
        return g.load().gllm_hip_kv_copy_rows_bytes(C.byref(a), C.byref(a), m.ctypes.data_as(C.c_void_p), len(m))

    def exchange(n):
        return moves((0, n, n), (n, 0, n))
    row = (1024 + 1024) * 2
    many = dict(layers=24, kd=1024, vd=1024)
    assert staged(exchange(40000), 80000, **many) == 80000 * row  # in order: one layer a launch, so all of its rows
    assert staged(exchange(32768), 65536, **many) == 65536 * row  # two
    assert staged(exchange(20000), 40000, **many) == 3 * 20000 * row  # three are enough
    shift = moves((5, 0, 5000))
    assert staged(shift, 5005, layers=32, kd=192, vd=192) == 0  # 32 layers of 6 workgroups
    assert staged(shift, 5005, layers=33, kd=192, vd=192) == 0  # and 17 of 6
    assert staged(shift, 5005, layers=32, kd=128, vd=128) == 0 and staged(shift, 5005, layers=33, kd=128, vd=128) == 17 * 5000 * 512
    # a launch's workspace is about 256 MB, whatever goes through it
    for n in (3000, 20000, 32768, 100000):
        for kw in (many, dict(layers=1, kd=64, vd=64), dict(layers=80, kd=256, vd=128)):
            layer = 2 * n * (kw["kd"] + kw["vd"]) * 2
            assert staged(exchange(n), 2 * n, **kw) <= max(256 << 20, layer)


def test_workspaces_over_the_tensors_are_refused():
    at = lambda x: C.c_void_p((1 << 20) + x)  # noqa: E731
    big = 1 << 30
    kv = cache(kd=256, vd=256)
    need, out = g.attend_tree_bytes(3, 4, 8, 2, 64, 10), 3 * 4 * 8 * 64 * 4
    tree = {**TREE, "kv": C.byref(kv), "q": at(0), "out": C.c_void_p(1 << 24)}
    for work in (at(0), at(16), at(out - 16), C.c_void_p((1 << 20) - need + 16), C.c_void_p((1 << 24) + out - 16)):
        refused("gllm_hip_attend_tree_dev", g.EINVAL, *{**tree, "work": work, "wb": big}.values())
        assert "overlap" in _lib.last_error()
    far = {**tree, "work": C.c_void_p(1 << 28), "wb": big}
    for name, size in (("starts", 12), ("lens", 12), ("parents", 48), ("counts", 12)):
        for shift in (0, need - 4, 4 - size):
            refused("gllm_hip_attend_tree_dev", g.EINVAL, *{**far, name: C.c_void_p((1 << 28) + shift)}.values())
            assert "overlap" in _lib.last_error()
    names = ("logits", "tokens", "parents", "counts", "path", "accepted", "next")
    apart = {**ACCEPT, **{n: C.c_void_p((i + 1) << 24) for i, n in enumerate(names)}}
    for n, size in zip(names, (((12 - 1) * 100 + 100) * 4, 48, 48, 12, 48, 12, 12)):
        for shift in (0, size // 16 * 16 - (size % 16 == 0) * 16):
            refused("gllm_hip_accept_tree_dev", g.EINVAL, *{**apart, "work": C.c_void_p(apart[n].value + shift), "wb": big}.values())
            assert "overlap" in _lib.last_error()


# --- the Python side ------------------------------------------------------------

PY_TREE = dict(layer=0, q=Tensor(3, 4, 512), n_heads=8, n_kv_heads=2, hd=64, starts=ints(3), lens=ints(3), most=10, parents=ints(3, 4),
               counts=ints(3), scale=0.1, out=Tensor(3, 4, 512))
PY_ACCEPT = dict(logits=Tensor(12, 100), tokens=ints(3, 4), parents=ints(3, 4), counts=ints(3), path=ints(3, 4), accepted=ints(3), next=ints(3))
PY_PATH = dict(starts=ints(3), lens=ints(3), path=ints(3, 4), accepted=ints(3))


def through(name, args):
    (api.accept_tree_dev if name == "accept_tree_dev" else getattr(py_cache(), name))(**args)


@pytest.mark.parametrize("name,args,wrong", [("attend_tree_dev", PY_TREE, w) for w in [
    dict(layer=FAR), dict(most=FAR), dict(q=Tensor(3, 4, 640)), dict(q=Tensor(3, 5, 512)), dict(q=Tensor(2, 4, 512)), dict(out=Tensor(3, 3, 512)),
    dict(out=Tensor(12, 8, 64)), dict(starts=ints(4)), dict(lens=ints(2)), dict(counts=ints(4)), dict(parents=ints(3, 5)), dict(parents=ints(12)),
    dict(parents=Tensor(3, 4)), dict(starts=Tensor(3)), dict(q=Tensor(3, 4, 512, device=1)), dict(lens=ints(3, 1)),
    dict(q=Tensor(3, 4, 512, strides=[4096, 1024, 1])), dict(work=Tensor(0, kind="uint8"))]] +
    [("accept_tree_dev", PY_ACCEPT, w) for w in [
        dict(logits=Tensor(11, 100)), dict(logits=Tensor(3, 4, 100)), dict(logits=Tensor(12, 100, strides=[100, 2])), dict(tokens=ints(3, 5)),
        dict(parents=ints(4, 4)), dict(counts=ints(4)), dict(path=ints(3, 3)), dict(accepted=ints(4)), dict(next=ints(2)),
        dict(tokens=Tensor(3, 4)), dict(path=Tensor(3, 4, kind="int32", strides=[8, 1])),
        dict(temperature=1.0, uniforms=Tensor(12)), dict(temperature=1.0, uniforms=ints(3, 4)), dict(logits=Tensor(12, 100, device=1)),
        dict(logits=Tensor(12, 100, strides=[FAR, 1]))]] +
    [("keep_path_dev", PY_PATH, w) for w in [dict(starts=ints(2)), dict(lens=ints(4)), dict(path=ints(12)), dict(accepted=ints(2)),
                                              dict(path=Tensor(3, 4)), dict(path=Tensor(3, 4, kind="int32", device=1))]])
def test_tensors_that_do_not_fit_are_refused(calls, name, args, wrong):  # noqa: F811
    through(name, args)
    assert len(calls) == 1  # as it is, the call gets through
    with pytest.raises(ValueError):
        through(name, {**args, **wrong})
    assert len(calls) == 1


def test_what_reaches_the_library(calls):  # noqa: F811
    through("attend_tree_dev", {**PY_TREE, "q": Tensor(12, 512), "counts": None})
    assert calls[0][0] == "gllm_hip_attend_tree_dev" and calls[0][4:9] == (3, 4, 8, 2, 64) and calls[0][13] is None
    through("accept_tree_dev", {**PY_ACCEPT, "logits": Tensor(12, 100, strides=[128, 1]), "temperature": 0.7, "uniforms": Tensor(3, 4)})
    assert calls[1][2:6] == (128, 100, 3, 4) and calls[1][9] == 0.7
    through("copy_rows_dev", dict(moves=[(1, 2, 3), (4, 5, 6)]))
    assert calls[2][4] == 2
    through("copy_rows_dev", dict(moves=[]))
    through("copy_rows_dev", dict(moves=np.array([[1, 2, 3]], np.int64)))
    assert [c[4] for c in calls[3:]] == [0, 1]
    for wrong in ([(1, 2)], [1, 2, 3], [(1, 2, FAR)], [(-FAR, 2, 3)], [(1.0, 2.0, 3.0)], np.zeros((2, 2, 3), int)):
        with pytest.raises(ValueError):
            through("copy_rows_dev", dict(moves=wrong))
    assert len(calls) == 5


def test_workspaces_past_32_bits_are_refused():
    for name, args in (("attend_tree_bytes", (1, 4, 8, 2, 64, FAR)), ("attend_tree_bytes", (FAR, 4, 8, 2, 64, 10)), ("accept_tree_bytes", (1, 4, FAR))):
        with pytest.raises(ValueError, match="32"):
            getattr(g, name)(*args)
