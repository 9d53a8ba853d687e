"""The cache operators on the device against their definitions in 64 bits:
rotary positions with the store, attention of a batch over a shared prefix and
own rows, attention that adds up the weight of every row, and the two ways to
give up rows.

Tolerances.  Scores: q carries 22 bits, products are exact, sums of hd terms
round at 2^-24 of their partial sums; with S = max scale * sum |q_d k_d| a
score is off by at most about S * (2^-22 + sqrt(hd) * 2^-23) and one more
rounding of the score, 2^-23 * S.  A weight is off by that relative to itself,
and by 2^-21 for the exponential and its own two parts.  Weighted means of
values up to V are then off by 2 V (those), and their sums add a like term:
u = 2 * (S * (2^-22 + (sqrt(hd) + 1) * 2^-23) + 2^-20).  f16 stores are exact
roundings, up to the float32 value next to a tie: half a step plus 2^-22.
"""
import math

import numpy as np
import pytest

from conftest import normal

pytestmark = pytest.mark.gpu

NAN = float("nan")


def cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


def make_cache(hip, rows, kd, seed, layers=1, vd=None, std=1.0, live=None):
    """A cache of N(0, std) rows; rows outside `live` hold NaN and infinities.
    Returns it with K and V as float64."""
    vd = vd or kd
    kv = hip.KVCacheF16(layers, kd, vd, rows)
    out = []
    for l in range(layers):
        k, v = normal(seed + 2 * l, (rows, kd), std).astype(np.float16), normal(seed + 2 * l + 1, (rows, vd)).astype(np.float16)
        if live is not None:
            dead = np.ones(rows, bool)
            for a, b in live:
                dead[max(a, 0):max(b, 0)] = False
            for x in (k, v):
                x[dead, 0::3], x[dead, 1::3], x[dead, 2::3] = np.nan, np.inf, -np.inf
        tk, tv = kv.tensors(l)
        tk.copy_(cuda(k))
        tv.copy_(cuda(v))
        out.append((k.astype(np.float64), v.astype(np.float64)))
    return (kv, *out[0]) if layers == 1 else (kv, out)


def attend64(q, k, v, rows, hd, n_kv, scale):
    """q (heads * hd) over the listed rows: (out, weights (heads, rows), bound on |out| errors per unit V)."""
    heads = q.size // hd
    r = heads // n_kv
    out, ws, s_max, v_max = np.zeros((heads, hd)), np.zeros((heads, len(rows))), 0.0, 0.0
    for h in range(heads):
        c = slice((h // r) * hd, (h // r) * hd + hd)
        if len(rows) == 0:
            continue
        qh = q[h * hd:(h + 1) * hd].astype(np.float64)
        s = k[rows, c] @ qh * scale
        s_max = max(s_max, float((np.abs(k[rows, c]) @ np.abs(qh)).max() * abs(scale)))
        w = np.exp(s - s.max())
        w /= w.sum()
        ws[h] = w
        out[h] = w @ v[rows, c]
        v_max = max(v_max, float(np.abs(v[rows, c]).max()))
    u = 2 * (s_max * (2.0 ** -22 + (math.sqrt(hd) + 1) * 2.0 ** -23) + 2.0 ** -20)
    return out.ravel(), ws, u, v_max


def check_shared(hip, n, heads, n_kv, hd, start, length, own, rows, seed, pad=0, std=1.0, scale=None, most=None, work=False):
    """own: [(start, len)] per request."""
    import torch
    live = [(start, start + length)] + [(a, a + max(m, 0)) for a, m in own]
    kv, k, v = make_cache(hip, rows, n_kv * hd + pad, seed, vd=n_kv * hd + 2 * pad, std=std, live=live)
    q = normal(seed + 9, (n, heads * hd))
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full((n, heads * hd), NAN, device="cuda")
    st = cuda(np.array([a for a, _ in own], np.int32)) if own else None
    ln = cuda(np.array([m for _, m in own], np.int32)) if own else None
    most = (max([1] + [m for _, m in own]) if own else 0) if most is None else most
    ws = torch.empty(hip.attend_shared_bytes(n, heads, n_kv, hd, length, most), dtype=torch.uint8, device="cuda") if work else None
    print(f"shared n {n} heads {heads}/{n_kv}x{hd} prefix {start}+{length} own {own[:4]} most {most}", flush=True)
    kv.attend_shared_dev(0, cuda(q), heads, n_kv, hd, start, length, st, ln, most, scale, out, work=ws)
    got = host(out)
    for i in range(n):
        at = list(range(start, start + length))
        if own:
            a, m = own[i]
            at += list(range(max(a, 0), min(rows, a + max(m, 0))))
        want, _, u, vm = attend64(q[i], k, v, np.array(at, int), hd, n_kv, scale)
        if not at:
            assert (got[i] == 0).all(), i
        assert np.isfinite(got[i]).all(), i
        assert np.abs(got[i] - want).max() <= u * vm + 1e-30, (i, np.abs(got[i] - want).max(), u * vm)


@pytest.mark.parametrize("n,heads,n_kv,hd,start,length,lens", [
    (1, 1, 1, 8, 0, 1, None),
    (1, 4, 1, 64, 3, 31, [1]),
    (2, 8, 2, 64, 0, 33, [0, 17]),
    (3, 32, 8, 128, 5, 130, [64, 0, 33]),
    (5, 40, 8, 80, 0, 257, [1, 2, 3, 0, 129]),       # 25 rows of a kv head
    (9, 10, 2, 40, 2, 1000, [32] * 9),                # 45 rows
    (17, 32, 8, 128, 0, 515, list(range(17))),        # 68 rows: two blocks
    (33, 32, 8, 128, 1, 700, [7] * 33),
    (3, 32, 1, 128, 0, 200, [40, 1, 300]),            # 32 query heads to one kv head
    (2, 71, 1, 64, 0, 100, [9, 70]),
    (4, 12, 12, 32, 0, 90, [5, 0, 1, 64]),
    (3, 6, 2, 96, 0, 0, [150, 0, 2]),                 # no prefix, one request with nothing
    (4, 4, 4, 24, 0, 0, None),                        # nothing at all
    (64, 8, 2, 16, 0, 40, [3] * 64),
])
def test_shared_prefix(hip, n, heads, n_kv, hd, start, length, lens):
    rows, own, at = start + length + 7, [], start + length + 3
    if lens:
        for m in lens:
            own.append((at, m))
            at += m
        rows = at + 5
    check_shared(hip, n, heads, n_kv, hd, start, length, own, rows, 100 + n + hd)


def test_shared_own_ranges_are_cut_to_the_cache(hip):
    check_shared(hip, 7, 8, 2, 64, 10, 20, [(-5, 9), (45, 100), (60, 3), (-4, 2), (30, -7), (2**31 - 1, 2**31 - 1), (0, 0)], 50, 300)


def test_shared_own_ranges_longer_than_planned(hip):
    check_shared(hip, 2, 8, 2, 64, 0, 10, [(10, 900), (500, 450)], 1000, 310, most=1)


def test_shared_several_tokens_of_a_request(hip):
    """Own ranges that start together and grow: causal tokens of one request."""
    check_shared(hip, 4, 8, 2, 128, 0, 64, [(64, 1), (64, 2), (64, 3), (64, 4)], 70, 320)


def test_shared_wider_cache_rows(hip):
    check_shared(hip, 3, 8, 2, 64, 0, 100, [(100, 5)] * 3, 110, 330, pad=24)


@pytest.mark.parametrize("std,scale", [(1e-4, None), (30.0, None), (1.0, 8.0), (1.0, 0.0), (1.0, -0.3), (6e-8, 1e4)])
def test_shared_score_ranges(hip, std, scale):
    """Keys from f16's least subnormals to large ones; scores from all equal to one row that takes it all."""
    check_shared(hip, 3, 8, 2, 64, 0, 300, [(300, 40)] * 3, 340, 340, std=std, scale=scale)


@pytest.mark.parametrize("mag", [1e-38, 1e-20, 1e18, 3e38])
def test_shared_query_magnitudes(hip, mag):
    """A query of any float32 size: scores are scaled back to size 1 through the scale."""
    import torch
    kv, k, v = make_cache(hip, 200, 128, 350)
    q = (normal(351, (1, 128)) / 4).astype(np.float64)
    qm = (q * mag).astype(np.float32)
    scale = float(np.float32(1 / mag)) if mag > 1e-30 else 1e37
    out = torch.empty((1, 128), device="cuda")
    kv.attend_shared_dev(0, cuda(qm), 2, 2, 64, 0, 200, None, None, 0, scale, out)
    want, _, u, vm = attend64(qm.astype(np.float64)[0], k, v, np.arange(200), 64, 2, scale)
    # a subnormal query has fewer bits, and so has a scale near the end of the range
    assert np.abs(host(out)[0] - want).max() <= u * vm * (64 if mag < 1e-37 or mag > 1e38 else 1)


@pytest.mark.parametrize("n,heads,n_kv,hd,length", [(40, 8, 2, 80, 45), (12, 8, 1, 72, 33), (3, 8, 2, 40, 70), (33, 16, 4, 120, 129), (64, 8, 2, 24, 1)])
def test_shared_reads_nothing_left_in_lds(hip, n, heads, n_kv, hd, length):
    """After a call that fills every LDS tile with NaN: head sizes and ranges that do not fill theirs."""
    import torch
    full = 128 if hd > 96 else 96 if hd > 64 else 64 if hd > 32 else 32
    kv = hip.KVCacheF16(1, 8 * full, 8 * full, 40000)
    for t in kv.tensors(0):
        t.fill_(NAN)
    out = torch.empty((n, heads // n_kv * 8 * full), device="cuda")
    kv.attend_shared_dev(0, torch.ones_like(out), heads // n_kv * 8, 8, full, 0, 40000, None, None, 0, 0.1, out)
    assert np.isnan(host(out)).all()
    check_shared(hip, n, heads, n_kv, hd, 2, length, [(length + 9, i % 3) for i in range(n)], length + 20, 355)


def test_shared_workspace_is_the_callers(hip):
    import torch
    check_shared(hip, 5, 8, 2, 64, 0, 300, [(300, 20)] * 5, 320, 360, work=True)
    kv, _, _ = make_cache(hip, 100, 128, 361)
    q, out = torch.zeros((2, 512), device="cuda"), torch.full((2, 512), 7.0, device="cuda")
    small = torch.empty(hip.attend_shared_bytes(2, 8, 2, 64, 100, 0) - 4, dtype=torch.uint8, device="cuda")
    with pytest.raises(hip.GllmError, match="workspace"):
        kv.attend_shared_dev(0, q, 8, 2, 64, 0, 100, None, None, 0, 0.1, out, work=small)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


def bound64(q, k, hd, scale):
    """The tolerance's u for float64 device tensors q (rows, hd) and k (positions, hd)."""
    s_max = float((q.abs() @ k.abs().T.contiguous()).max()) * abs(scale)
    return 2 * (s_max * (2.0 ** -22 + (math.sqrt(hd) + 1) * 2.0 ** -23) + 2.0 ** -20)


# enough work for 32 query rows a wave: over 4e9 rows x positions x head size
@pytest.mark.parametrize("n,r,hd,length", [(1024, 8, 128, 4001), (2048, 8, 80, 3201), (2048, 8, 40, 6503), (2048, 8, 24, 10901), (63, 65, 128, 7815)])
def test_shared_many_rows_over_long_prefixes(hip, n, r, hd, length):
    import torch
    most = 3
    kv, k, v = make_cache(hip, length + most * n + 1, hd, 375)
    q = normal(376, (n, r * hd))
    starts = cuda((length + most * np.arange(n)).astype(np.int32))
    lens = cuda((np.arange(n) % (most + 1)).astype(np.int32))
    out = torch.empty((n, r * hd), device="cuda")
    print(f"shared, many rows: {n} x {r} x {hd} over {length}", flush=True)
    kv.attend_shared_dev(0, cuda(q), r, 1, hd, 0, length, starts, lens, most, hd ** -0.5, out)
    q64, k64, v64 = cuda(q).double().view(n, r, hd), cuda(k), cuda(v)
    rows = starts.long()[:, None] + torch.arange(most, device="cuda")
    s = torch.cat([(q64.view(-1, hd) @ k64[:length].T.contiguous()).view(n, r, length), (q64[:, :, None] * k64[rows][:, None]).sum(-1)], -1) * hd ** -0.5
    s[..., length:].masked_fill_((torch.arange(most, device="cuda") >= lens[:, None])[:, None], -math.inf)
    w = torch.softmax(s, -1)
    want = (w[..., :length].reshape(-1, length) @ v64[:length]).view(n, r, hd) + (w[..., length:, None] * v64[rows][:, None]).sum(2)
    u = bound64(q64.view(-1, hd), k64, hd, hd ** -0.5)
    assert float((out.double().view(n, r, hd) - want).abs().max()) <= u * float(v64.abs().max())


def test_mass_many_rows_over_a_long_prefix(hip):
    import torch
    n, r, hd, length = 1024, 8, 128, 5200
    kv, k, v = make_cache(hip, length, hd, 377)
    q = normal(378, (n, r * hd))
    out, mass = torch.empty((n, r * hd), device="cuda"), torch.zeros((1, length), device="cuda")
    print("mass, many rows", flush=True)
    kv.attend_mass_dev(0, cuda(q), r, 1, hd, 0, length - 1, hd ** -0.5, mass, out)
    q64, k64, v64 = cuda(q).double().view(-1, hd), cuda(k), cuda(v)
    s = (q64 @ k64.T.contiguous()).view(n, r, length) * hd ** -0.5
    s.masked_fill_((torch.arange(length, device="cuda") > length - n + torch.arange(n, device="cuda")[:, None])[:, None], -math.inf)
    w = torch.softmax(s, -1)
    want, per = w.view(-1, length) @ v64, w.sum((0, 1))
    u = bound64(q64, k64, hd, hd ** -0.5)
    assert float((out.double().view(-1, hd) - want).abs().max()) <= u * float(v64.abs().max())
    # n * r additions, tile by tile: at most as many roundings as the sum has terms
    assert bool(((mass[0].double() - per).abs() <= (u + n * r * 2.0 ** -24) * per).all())


def test_shared_agrees_with_the_single_sequence(hip):
    """n equal requests over a prefix are n times attend_dev over the same rows."""
    import torch
    kv, k, v = make_cache(hip, 500, 1024, 370)
    q = normal(371, (1, 4096))
    out, one = torch.empty((6, 4096), device="cuda"), torch.empty(4096, device="cuda")
    kv.attend_shared_dev(0, cuda(np.repeat(q, 6, 0)), 32, 8, 128, 2, 490, None, None, 0, 128 ** -0.5, out)
    kv.attend_dev(0, cuda(q), 32, 8, 128, 2, 491, 128 ** -0.5, one)
    got = host(out)
    assert (got == got[0]).all()
    _, _, u, vm = attend64(q[0], k, v, np.arange(2, 492), 128, 8, 128 ** -0.5)
    assert np.abs(got[0] - host(one)).max() <= 2 * u * vm


def test_shared_long_cache_past_32_bit_offsets(hip):
    """Rows whose byte offset in K and V passes 4 GiB, and whose element offset passes 2^31."""
    import torch
    rows, dim = 1_100_000, 2048
    kv = hip.KVCacheF16(1, dim, dim, rows)
    a, m = rows - 333, 333
    k, v = normal(380, (m, dim)).astype(np.float16), normal(381, (m, dim)).astype(np.float16)
    tk, tv = kv.tensors(0)
    tk[a:].copy_(cuda(k))
    tv[a:].copy_(cuda(v))
    q = normal(382, (2, 2048))
    out = torch.empty((2, 2048), device="cuda")
    print("shared: far rows", flush=True)
    kv.attend_shared_dev(0, cuda(q), 16, 16, 128, a, 300, cuda(np.array([rows - 33, rows - 1], np.int32)),
                         cuda(np.array([33, 1], np.int32)), 33, 128 ** -0.5, out)
    got = host(out)
    k64, v64 = k.astype(np.float64), v.astype(np.float64)
    for i, at in enumerate((np.arange(333), np.r_[np.arange(300), 332])):
        want, _, u, vm = attend64(q[i], k64, v64, at, 128, 16, 128 ** -0.5)
        assert np.abs(got[i] - want).max() <= u * vm


def test_shared_on_another_stream_and_in_two_graphs(hip):
    """Two graphs with workspaces of their own, captured on one stream, replayed at once on two streams,
    with other work between the replays; lengths change under the graphs."""
    import torch
    kv, k, v = make_cache(hip, 800, 256, 390)
    qs = [normal(391 + i, (4, 512)) for i in range(2)]
    dq = [cuda(q) for q in qs]
    starts = cuda(np.array([400, 500, 600, 700], np.int32))
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")
    outs = [torch.empty((4, 512), device="cuda") for _ in range(2)]
    wb = hip.attend_shared_bytes(4, 8, 4, 64, 400, 100)
    works = [torch.empty(wb, dtype=torch.uint8, device="cuda") for _ in range(2)]
    side, graphs = torch.cuda.Stream(), []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kv.attend_shared_dev(0, dq[i], 8, 4, 64, 0, 400, starts, lens, 100, 0.125, outs[i], work=works[i])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for m in (0, 1, 57, 100):
        lens.fill_(m)
        for o in outs:
            o.fill_(NAN)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            got = host(outs[i])
            for t in range(4):
                at = np.r_[np.arange(400), 400 + 100 * t + np.arange(m)]
                want, _, u, vm = attend64(qs[i][t], k, v, at, 64, 4, 0.125)
                assert np.abs(got[t] - want).max() <= u * vm, (m, i, t)


# --- the weight of every row ----------------------------------------------------


@pytest.mark.parametrize("n,heads,n_kv,hd,start,end", [
    (1, 1, 1, 8, 0, 0), (1, 32, 8, 128, 0, 40), (1, 8, 2, 64, 5, 700), (3, 8, 2, 64, 0, 2), (16, 32, 8, 128, 3, 200),
    (7, 10, 2, 80, 0, 301), (33, 8, 4, 32, 0, 33), (40, 4, 1, 96, 0, 1000), (32, 32, 8, 128, 0, 600), (1, 71, 1, 128, 0, 130),
])
def test_mass(hip, n, heads, n_kv, hd, start, end):
    import torch
    rows = end + 4
    kv, k, v = make_cache(hip, rows, n_kv * hd, 500 + n + hd, live=[(start, end + 1)])
    q = normal(501, (n, heads * hd))
    before = np.abs(normal(502, (n_kv, rows + 3)))
    mass, out = cuda(before), torch.full((n, heads * hd), NAN, device="cuda")
    print(f"mass n {n} heads {heads}/{n_kv}x{hd} rows {start}..{end}", flush=True)
    kv.attend_mass_dev(0, cuda(q), heads, n_kv, hd, start, end, hd ** -0.5, mass, out)
    got, got_mass = host(out), host(mass)
    want_mass, total = before.astype(np.float64), 0.0
    slack = np.zeros_like(want_mass)
    for i in range(n):
        at = np.arange(start, end - (n - 1) + i + 1)
        want, w, u, vm = attend64(q[i], k, v, at, hd, n_kv, hd ** -0.5)
        assert np.abs(got[i] - want).max() <= u * vm, i
        per = w.reshape(n_kv, heads // n_kv, -1).sum(1)
        want_mass[:, at] += per
        slack[:, at] += u * per
        total += heads
    live = np.zeros(rows + 3, bool)
    live[start:end + 1] = True
    assert np.array_equal(got_mass[:, ~live], before[:, ~live])
    # the sum's own roundings: n * r additions and the one onto what was there
    slack += (n * heads // n_kv + 2) * 2.0 ** -24 * want_mass
    assert (np.abs(got_mass - want_mass) <= slack + 1e-30).all()
    assert abs((got_mass - before)[:, live].sum() - total) <= 1e-4 * total + 1e-5 * rows


@pytest.mark.parametrize("n,heads,n_kv,hd,end", [(3, 2, 1, 64, 50), (4, 8, 2, 128, 31), (20, 8, 2, 128, 65), (40, 4, 1, 96, 130), (5, 2, 2, 40, 4)])
def test_mass_rows_that_only_later_tokens_see(hip, n, heads, n_kv, hd, end):
    """Infinities and NaN in the last tokens' own rows stay out of the tokens before."""
    kv, k, v = make_cache(hip, end + 3, n_kv * hd, 530, live=[(0, end - 1)])  # the last two tokens' rows are not finite
    import torch
    q, out = normal(531, (n, heads * hd)), torch.empty((n, heads * hd), device="cuda")
    mass = torch.zeros((n_kv, end + 1), device="cuda")
    print(f"mass, later rows not finite: n {n} heads {heads}/{n_kv}x{hd} end {end}", flush=True)
    kv.attend_mass_dev(0, cuda(q), heads, n_kv, hd, 0, end, hd ** -0.5, mass, out)
    got = host(out)
    for i in range(n - 2):
        want, _, u, vm = attend64(q[i], k, v, np.arange(end - (n - 1) + i + 1), hd, n_kv, hd ** -0.5)
        assert np.abs(got[i] - want).max() <= u * vm, i


def test_capture_without_a_workspace_needs_an_earlier_call(hip):
    """The library's scratch does not grow under capture: the call is refused and captures nothing."""
    import torch
    kv, _, _ = make_cache(hip, 5000, 128, 540)
    q, out = torch.zeros((2, 512), device="cuda"), torch.full((2, 512), 7.0, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph, stream=side):
        x.add_(1.0)
        with pytest.raises(hip.GllmError) as e:
            kv.attend_shared_dev(0, q, 8, 2, 64, 0, 5000, None, None, 0, 0.1, out)
        assert e.value.code == hip.EUNSUP
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 7.0).all() and (x == 1.0).all()
    hip.stream_release(side.cuda_stream)


def test_two_host_threads_at_once(hip):
    """Calls of two threads on two streams over one cache, each with the library's scratch of its own."""
    import threading
    import torch
    kv, k, v = make_cache(hip, 900, 256, 550)
    qs = [normal(551 + i, (9, 512)) for i in range(2)]
    wants = [[attend64(q[t], k, v, np.arange(900), 64, 4, 0.125) for t in range(9)] for q in qs]
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            dq, out = cuda(qs[i]), torch.empty((9, 512), device="cuda")
            for _ in range(20):
                kv.attend_shared_dev(0, dq, 8, 4, 64, 0, 900, None, None, 0, 0.125, out)
            s.synchronize()
            got = out.cpu().numpy()
        for t, (want, _, u, vm) in enumerate(wants[i]):
            if not np.abs(got[t] - want).max() <= u * vm:
                bad.append((i, t))
        hip.stream_release(s.cuda_stream)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_mass_adds_up_over_calls_and_replays(hip):
    """Two eager calls and three replays of a captured one add five times the weights."""
    import torch
    kv, k, v = make_cache(hip, 300, 256, 520)
    q = normal(521, (2, 512))
    dq, out = cuda(q), torch.empty((2, 512), device="cuda")
    mass = torch.zeros((4, 300), device="cuda")
    work = torch.empty(hip.attend_mass_bytes(2, 8, 4, 64, 300), dtype=torch.uint8, device="cuda")
    call = lambda: kv.attend_mass_dev(0, dq, 8, 4, 64, 0, 299, 0.125, mass, out, work=work)  # noqa: E731
    call()
    one = host(mass).astype(np.float64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    call()
    for _ in range(3):
        graph.replay()
        torch.zeros(1000, device="cuda").add_(1.0)
        torch.cuda.synchronize()
    assert np.allclose(host(mass), 5 * one, rtol=2.0 ** -21, atol=0)


# --- rotary positions -------------------------------------------------------------


def rotate64(x, pos, inv, amp, hd, half):
    x = x.reshape(x.shape[0], -1, hd).astype(np.float64)
    rot = 2 * len(inv)
    ang = pos.astype(np.float64)[:, None] * inv
    c, s = (np.cos(ang) * amp)[:, None], (np.sin(ang) * amp)[:, None]
    y = x.copy()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y.reshape(x.shape[0], -1)


ROPES = [
    (1, 32, 8, 128, dict()), (3, 8, 2, 64, dict(layout="half")), (7, 5, 5, 80, dict(rot_dim=32)),
    (65, 4, 1, 96, dict(layout="half", rot_dim=48, scaling="yarn", factor=8.0, orig_ctx=2048)),
    (2, 3, 1, 8, dict(rot_dim=2)), (300, 4, 2, 128, dict(scaling="llama3", factor=8.0, orig_ctx=8192)),
    (9, 2, 1, 50, dict(rot_dim=26, scaling="linear", factor=3.0, attn_factor=0.5)),
    (4, 2, 2, 66, dict(rot_dim=66, layout="half", freq_factors=np.linspace(1, 4, 33, dtype=np.float32))),
    (5, 1, 1, 1024, dict(theta=10000.0)), (2, 300, 2, 1024, dict(layout="half")), (3, 6, 2, 64, dict(rot_dim=20, layout="half")),
]


def rope_positions(n, seed):
    pos = np.random.default_rng(seed).integers(0, 1 << 20, n).astype(np.int32)
    pos[0] = 0
    pos[-1] = 2**31 - 1
    if n > 2:
        pos[1] = -(2**31)
    return pos


@pytest.mark.parametrize("n,heads,n_kv,hd,kw", ROPES)
def test_rope_and_store(hip, n, heads, n_kv, hd, kw):
    import torch
    rope = hip.Rope(hd, **kw)
    inv, amp = hip.Rope.frequencies(hd, **kw)
    half = kw.get("layout") == "half"
    rows = n + 6
    kv = hip.KVCacheF16(2, n_kv * hd + 8, n_kv * hd + 16, rows)
    fused = normal(600 + n, (n, (heads + 2 * n_kv) * hd + 3))  # rows of q, k, v and something else
    q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + n_kv) * hd], fused[:, (heads + n_kv) * hd:(heads + 2 * n_kv) * hd]
    pos = rope_positions(n, 601)
    at = np.random.default_rng(602).permutation(rows)[:n].astype(np.int32)
    stored = np.ones(n, bool)
    if n > 4:
        at[2], at[3], stored[2:4] = -1, rows, False
    before = [[normal(603 + 2 * l + j, (rows, d)).astype(np.float16) for j, d in enumerate((n_kv * hd + 8, n_kv * hd + 16))] for l in range(2)]
    for l in range(2):
        for t, b in zip(kv.tensors(l), before[l]):
            t.copy_(cuda(b))
    f = cuda(fused)
    out = torch.full((n, heads * hd + 5), NAN, device="cuda")
    print(f"rope n {n} heads {heads}/{n_kv}x{hd} {kw}", flush=True)
    kv.store_rope_dev(1, rope, f[:, :heads * hd], f[:, heads * hd:(heads + n_kv) * hd],
                      f[:, (heads + n_kv) * hd:(heads + 2 * n_kv) * hd], cuda(pos), cuda(at), out[:, :heads * hd])
    got = host(out)
    # c, s and the products round once each: 2^-24 of either product, and the sum once
    tol = 4 * 2.0 ** -24 * amp * np.abs(q).max() + 1e-30
    assert np.abs(got[:, :heads * hd] - rotate64(q, pos, inv, amp, hd, half)).max() <= tol
    assert np.isnan(got[:, heads * hd:]).all()
    wk = rotate64(k, pos, inv, amp, hd, half)
    K, V = (host(t) for t in kv.tensors(1))
    dk = n_kv * hd
    for t in range(n):
        if stored[t]:
            err = np.abs(K[at[t], :dk].astype(np.float64) - wk[t])
            assert (err <= np.maximum(np.abs(wk[t]) * 2.0 ** -11, 2.0 ** -25) + tol).all(), t
            assert np.array_equal(V[at[t], :dk], v[t].astype(np.float16))
    other = np.ones(rows, bool)
    other[at[stored]] = False
    for x, b in ((K, before[1][0]), (V, before[1][1])):
        assert np.array_equal(x[other], b[other]) and np.array_equal(x[:, dk:], b[:, dk:])
    for t, b in zip(kv.tensors(0), before[0]):
        assert np.array_equal(host(t), b)


@pytest.mark.parametrize("n,heads,n_kv,hd,kw", ROPES)
def test_rope_alone_and_in_place(hip, n, heads, n_kv, hd, kw):
    import torch
    rope = hip.Rope(hd, **kw)
    inv, amp = hip.Rope.frequencies(hd, **kw)
    x, pos = normal(620, (n, heads * hd)), rope_positions(n, 621)
    want = rotate64(x, pos, inv, amp, hd, kw.get("layout") == "half")
    tol = 4 * 2.0 ** -24 * amp * np.abs(x).max()
    t = cuda(x)
    out = rope.apply_dev(t, cuda(pos), torch.empty_like(t))
    assert np.abs(host(out) - want).max() <= tol and np.array_equal(host(t), x)
    rope.apply_dev(t, cuda(pos))
    assert np.array_equal(host(t), host(out))


def test_rope_turns_as_the_decoder_does(hip):
    """Interleaved rotation at small positions, where the decoder's float32 angle is exact enough."""
    from oracle import oracle as ref
    x = normal(630, (1, 512))
    inv = ref.rope_inv_freq(500000.0, 64)
    s, c = ref.rope_sincos(3, inv)
    want = ref.rope_apply(x[0], 64, 8, s, c)
    t = cuda(x)
    hip.Rope(64).apply_dev(t, cuda(np.array([3], np.int32)))
    # the decoder's frequencies and angle are float32: 2 roundings of an angle up to 3
    assert np.abs(host(t)[0] - want).max() <= np.abs(x).max() * (3 * 2 * 2.0 ** -24 + 6 * 2.0 ** -24)


def test_rope_in_quads_and_strided(hip):
    """Aligned rows of a fused projection (quads) against the same values one row off (pairs)."""
    import torch
    rope = hip.Rope(64, rot_dim=32, layout="half")
    x = cuda(normal(640, (9, 3 * 64 + 8)))
    pos = cuda(rope_positions(9, 641))
    quads = rope.apply_dev(x[:, :192], pos, torch.empty((9, 192), device="cuda"))
    odd = torch.empty((9, 3 * 64 + 7), device="cuda")
    odd[:, 1:193].copy_(x[:, :192])
    pairs = rope.apply_dev(odd[:, 1:193], pos, torch.empty((9, 193), device="cuda")[:, 1:])
    assert np.array_equal(host(quads), host(pairs))


def test_rope_no_tokens_and_refusals(hip):
    import torch
    rope = hip.Rope(64)
    kv = hip.KVCacheF16(1, 128, 128, 10)
    none = torch.zeros((0, 128), device="cuda")
    ints = torch.zeros(0, dtype=torch.int32, device="cuda")
    rope.apply_dev(none, ints)
    kv.store_rope_dev(0, rope, none, none, none, ints, ints)
    x, pos = torch.zeros((3, 128), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (lambda: rope.apply_dev(x[:, :100], pos), lambda: rope.apply_dev(x.double(), pos), lambda: rope.apply_dev(x.T, pos),
                lambda: rope.apply_dev(x, pos.long()), lambda: rope.apply_dev(x[:2], pos), lambda: rope.apply_dev(x.cpu(), pos),
                lambda: rope.apply_dev(x, pos.cpu()), lambda: rope.apply_dev(x, pos, x[:1].expand(3, 128)),
                lambda: kv.store_rope_dev(0, rope, x, x, x[:, :64], pos, pos)):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros((3, 256), device="cuda")
    for bad in (lambda: kv.store_rope_dev(1, rope, x, x, x, pos, pos), lambda: kv.store_rope_dev(0, rope, x, wide, wide, pos, pos)):
        with pytest.raises(hip.GllmError):
            bad()


# --- giving up rows -----------------------------------------------------------------


def order_of(mass, pos, sinks, frm):
    """Rows best first: protected ones (all alike), then by mass, NaN last, ties to the lowest row."""
    stay = (pos < sinks) | (pos >= frm)
    num = np.where(np.isnan(mass), -np.inf, mass.astype(np.float64))
    num, nan = np.where(stay, 0, num), np.isnan(mass) & ~stay
    return np.lexsort((np.arange(len(mass)), -num, nan, ~stay))


def masses(seed, shape):
    """Heavy-tailed weights with equal values, zeros of both signs, infinities and NaN."""
    rng = np.random.default_rng(seed)
    m = (rng.random(shape) ** 8).astype(np.float32)
    m[rng.random(shape) < 0.3] = np.float32(0.25)
    for x, p in ((0.0, 0.05), (-0.0, 0.05), (np.inf, 0.01), (-np.inf, 0.01), (np.nan, 0.02), (-1.5, 0.02), (1e-42, 0.02)):
        m[rng.random(shape) < p] = x
    return m


@pytest.mark.parametrize("layers,n_kv,hd,start,length,dst_start,budget,sinks,recent,with_pos", [
    (1, 1, 8, 0, 1, 0, 1, 0, 0, False), (2, 2, 64, 3, 50, 2, 20, 4, 5, True), (1, 8, 128, 0, 1025, 0, 300, 0, 0, False),
    (3, 3, 40, 1, 2500, 0, 2500, 4, 100, True), (1, 2, 32, 0, 700, 5, 1, 2, 3, True), (1, 1, 16, 0, 5000, 0, 4999, 0, 64, False),
    (1, 1, 8, 0, 4096, 0, 700, 4, 9, True), (1, 2, 8, 0, 16385, 0, 9000, 4, 9, True), (1, 1, 8, 3, 65536, 0, 30000, 0, 100, False),
    (1, 2, 8, 0, 65537, 0, 20000, 4, 64, True), (1, 1, 8, 0, 140001, 1, 139000, 4, 64, True), (1, 1, 8, 0, 100000, 0, 1, 0, 0, True),
    (40, 1, 8, 0, 90, 0, 30, 1, 9, True), (1, 2, 64, 0, 300, 0, 50, 100, 100, True), (1, 2, 64, 0, 6000, 0, 1000, 0, 0, True),
])
def test_keep(hip, layers, n_kv, hd, start, length, dst_start, budget, sinks, recent, with_pos):
    import torch
    rows, out_rows = start + length + 2, dst_start + budget + 3
    dim = n_kv * hd
    src, dst = hip.KVCacheF16(layers, dim + 8, dim, rows), hip.KVCacheF16(layers, dim, dim + 16, out_rows)
    data = [[normal(700 + 2 * l + j, (rows, d)).astype(np.float16) for j, d in enumerate((dim + 8, dim))] for l in range(layers)]
    for l in range(layers):
        for t, b in zip(src.tensors(l), data[l]):
            t.copy_(cuda(b))
    mass = masses(701, (layers, n_kv, rows + 1))
    if layers == 1 and length == 6000:
        mass[:] = 0.5  # every row ties
    rng = np.random.default_rng(702)
    pos = np.stack([[rng.permutation(rows + 1) for _ in range(n_kv)] for _ in range(layers)]).astype(np.int32)
    now = rows + 1
    mass_out = torch.full((layers, n_kv, out_rows), NAN, device="cuda")
    pos_out = torch.full((layers, n_kv, out_rows), -7, dtype=torch.int32, device="cuda")
    print(f"keep {budget} of {start}+{length}, {layers}x{n_kv}x{hd}", flush=True)
    src.keep_dev(dst, n_kv, hd, length, budget, cuda(mass), cuda(pos) if with_pos else None, mass_out, pos_out, now=now,
                 sinks=sinks, recent=recent, start=start, dst_start=dst_start)
    got_m, got_p = host(mass_out), host(pos_out)
    inside = np.zeros(out_rows, bool)
    inside[dst_start:dst_start + budget] = True
    assert np.isnan(got_m[:, :, ~inside]).all() and (got_p[:, :, ~inside] == -7).all()
    for l in range(layers):
        tk, tv = (host(t) for t in dst.tensors(l))
        assert (tk[~inside] == 0).all() and (tv[~inside] == 0).all() and (tv[:, dim:] == 0).all()
        for g in range(n_kv):
            p = (pos[l, g] if with_pos else np.arange(rows + 1))[start:start + length]
            best = order_of(mass[l, g, start:start + length], p, sinks, now - recent)
            keep = np.sort(best[:budget])
            assert np.array_equal(got_p[l, g, inside], p[keep]), (l, g)
            assert np.array_equal(got_m[l, g, inside].view(np.uint32), mass[l, g, start + keep].view(np.uint32))
            c = slice(g * hd, g * hd + hd)
            assert np.array_equal(tk[inside, c], data[l][0][start + keep, c]) and np.array_equal(tv[inside, c], data[l][1][start + keep, c])


@pytest.mark.parametrize("n_kv,hd,start,length,sinks,recent", [
    (1, 8, 0, 1, 0, 0), (8, 128, 0, 1024, 4, 32), (3, 40, 5, 700, 0, 0), (2, 64, 0, 1500, 2000, 0), (5, 80, 2, 5000, 4, 5000), (2, 1, 0, 40, 1, 1)])
def test_evict_and_store(hip, n_kv, hd, start, length, sinks, recent):
    import torch
    rows, dim = start + length + 3, n_kv * hd
    kv = hip.KVCacheF16(2, dim + 3, dim, rows)
    data = [normal(800 + j, (rows, d)).astype(np.float16) for j, d in enumerate((dim + 3, dim))]
    for t, b in zip(kv.tensors(1), data):
        t.copy_(cuda(b))
    mass = masses(801, (n_kv, rows + 2))
    mass[:, start:start + length][mass[:, start:start + length] < 0] = 0.125
    mass[np.isnan(mass) | np.isinf(mass)] = 0.5  # from the second call on the victim has to be new
    rng = np.random.default_rng(802)
    pos = np.stack([rng.permutation(rows + 2) for _ in range(n_kv)]).astype(np.int32)
    dm, dp = cuda(mass), cuda(pos)
    now = torch.zeros(1, dtype=torch.int32, device="cuda")
    victims = torch.full((n_kv,), -1, dtype=torch.int32, device="cuda")
    for step in range(3):
        at = rows + 2 + step
        k, v = normal(803 + step, dim), normal(813 + step, dim)
        now.fill_(at)
        print(f"evict {n_kv}x{hd} of {start}+{length}, step {step}", flush=True)
        kv.evict_store_dev(1, n_kv, hd, cuda(k), cuda(v), start, length, dm, dp, now, sinks=sinks, recent=recent, rows_out=victims)
        got = host(victims)
        for g in range(n_kv):
            m, p = mass[g, start:start + length], pos[g, start:start + length]
            stay = (p < sinks) | (p >= at - recent)
            t = int(np.lexsort((np.arange(length), np.where(stay, 0, m), stay))[0]) + start
            assert got[g] == t, (step, g)
            mass[g, t], pos[g, t] = 0.0, at
            c = slice(g * hd, g * hd + hd)
            data[0][t, c], data[1][t, c] = k[c].astype(np.float16), v[c].astype(np.float16)
        assert np.array_equal(host(dm), mass) and np.array_equal(host(dp), pos)
        for t, b in zip(kv.tensors(1), data):
            assert np.array_equal(host(t), b)
    for t in kv.tensors(0):
        assert (host(t) == 0).all()


def test_evict_gives_up_nan_first(hip):
    import torch
    kv = hip.KVCacheF16(1, 8, 8, 70)
    mass = np.full((1, 70), -np.inf, np.float32)
    mass[0, 66] = np.nan
    pos = cuda(np.arange(70, dtype=np.int32)[None])
    victims = torch.zeros(1, dtype=torch.int32, device="cuda")
    z = torch.zeros(8, device="cuda")
    kv.evict_store_dev(0, 1, 8, z, z, 0, 70, cuda(mass), pos, torch.tensor([99], dtype=torch.int32, device="cuda"), rows_out=victims)
    assert host(victims)[0] == 66


def test_far_rows_of_a_long_cache(hip):
    """Store, weights, keeping and evicting at rows past 4 GiB of K and of V (and 2^31 values)."""
    import torch
    rows, n_kv, hd = 1_100_000, 16, 128
    dim = n_kv * hd
    kv, small = hip.KVCacheF16(1, dim, dim, rows), hip.KVCacheF16(1, dim, dim, 10)
    n = 40
    a = rows - n
    rope = hip.Rope(hd)
    inv, amp = hip.Rope.frequencies(hd)
    k, v = normal(850, (n, dim)), normal(851, (n, dim))
    pos = np.arange(n, dtype=np.int32)
    print("far rows: store", flush=True)
    kv.store_rope_dev(0, rope, None, cuda(k), cuda(v), cuda(pos), cuda((a + pos).astype(np.int32)))
    tk, tv = kv.tensors(0)
    k16, v16 = host(tk[a:]), host(tv[a:])
    assert np.abs(k16 - rotate64(k, pos, inv, amp, hd, False)).max() <= np.abs(k).max() * 2.0 ** -10
    assert np.array_equal(v16, v.astype(np.float16)) and not host(tk[:n]).any() and not host(tv[:n]).any()
    k64, v64 = k16.astype(np.float64), v16.astype(np.float64)
    for tokens in (1, 3):  # scores kept, and made again
        q, out = normal(852, (tokens, 2 * dim)), torch.empty((tokens, 2 * dim), device="cuda")
        mass = torch.zeros((n_kv, rows), device="cuda")
        print(f"far rows: weights of {tokens}", flush=True)
        kv.attend_mass_dev(0, cuda(q), 2 * n_kv, n_kv, hd, a, rows - 1, hd ** -0.5, mass, out)
        got, want = host(mass), np.zeros((n_kv, n))
        for i in range(tokens):
            at = np.arange(n - tokens + i + 1)
            o, w, u, vm = attend64(q[i], k64, v64, at, hd, n_kv, hd ** -0.5)
            want[:, at] += w.reshape(n_kv, 2, -1).sum(1)
            assert np.abs(host(out)[i] - o).max() <= u * vm
        assert np.abs(got[:, a:] - want).max() <= (u + 2.0 ** -20) * want.max() and not got[:, :a].any()
    m2, p2 = torch.zeros((1, n_kv, 10), device="cuda"), torch.zeros((1, n_kv, 10), dtype=torch.int32, device="cuda")
    print("far rows: keep", flush=True)
    kv.keep_dev(small, n_kv, hd, n, 10, mass[None], None, m2, p2, now=rows, start=a)
    sk = host(small.tensors(0)[0])
    for g in range(n_kv):
        best = np.sort(order_of(got[g, a:], np.arange(a, rows), 0, rows)[:10])
        assert np.array_equal(host(p2)[0, g], a + best) and np.array_equal(sk[:, g * hd:g * hd + hd], k16[best, g * hd:g * hd + hd])
    positions = torch.arange(rows, dtype=torch.int32, device="cuda").repeat(n_kv, 1)
    gone, now = torch.zeros(n_kv, dtype=torch.int32, device="cuda"), torch.full((1,), rows, dtype=torch.int32, device="cuda")
    print("far rows: evict", flush=True)
    kv.evict_store_dev(0, n_kv, hd, cuda(k[0]), cuda(v[0]), a, n, mass, positions, now, rows_out=gone)
    for g in range(n_kv):
        t = int(np.argmin(got[g, a:]))
        assert host(gone)[g] == a + t
        assert np.array_equal(host(tv[a + t])[g * hd:g * hd + hd], v[0, g * hd:g * hd + hd].astype(np.float16))


# --- a run of them together ------------------------------------------------------------


def test_a_bounded_cache_from_prompt_to_decode(hip):
    """Prompt rows rotated and stored, the last tokens' weights, down to a budget, then decode steps that
    track weights and replace rows: against the same steps in 64 bits on the device's own choices."""
    import torch
    heads, n_kv, hd, prompt, window, budget, sinks, recent = 8, 2, 64, 400, 16, 96, 4, 16
    dim, scale = n_kv * hd, hd ** -0.5
    rope = hip.Rope(hd, layout="half", scaling="llama3", factor=8.0, orig_ctx=256)
    inv, amp = hip.Rope.frequencies(hd, layout="half", scaling="llama3", factor=8.0, orig_ctx=256)
    big, small = hip.KVCacheF16(1, dim, dim, prompt), hip.KVCacheF16(1, dim, dim, budget)
    x = normal(900, (prompt + 6, heads * hd + 2 * dim))
    dx = cuda(x)
    pos = torch.arange(prompt + 6, dtype=torch.int32, device="cuda")
    parts = lambda a, b: (dx[a:b, :heads * hd], dx[a:b, heads * hd:heads * hd + dim], dx[a:b, heads * hd + dim:])  # noqa: E731
    q = torch.empty((prompt, heads * hd), device="cuda")
    qs, ks, vs = parts(0, prompt)
    big.store_rope_dev(0, rope, qs, ks, vs, pos[:prompt], pos[:prompt], q)
    mass, out = torch.zeros((1, n_kv, prompt), device="cuda"), torch.empty((window, heads * hd), device="cuda")
    big.attend_mass_dev(0, q[-window:], heads, n_kv, hd, 0, prompt - 1, scale, mass[0], out)
    m2 = torch.zeros((1, n_kv, budget), device="cuda")
    p2 = torch.zeros((1, n_kv, budget), dtype=torch.int32, device="cuda")
    big.keep_dev(small, n_kv, hd, prompt, budget, mass, None, m2, p2, now=prompt, sinks=sinks, recent=recent)
    # the same in 64 bits
    q64, k64 = (rotate64(x[:, a:b], np.arange(prompt + 6), inv, amp, hd, True) for a, b in ((0, heads * hd), (heads * hd, heads * hd + dim)))
    k16, v16 = k64.astype(np.float16).astype(np.float64), x[:, heads * hd + dim:].astype(np.float16).astype(np.float64)
    want = np.zeros((n_kv, prompt))
    for i in range(window):
        at = np.arange(prompt - window + i + 1)
        o, w, _, _ = attend64(q64[prompt - window + i], k16, v16, at, hd, n_kv, scale)
        want[:, at] += w.reshape(n_kv, heads // n_kv, -1).sum(1)
        assert np.abs(host(out)[i] - o).max() <= 2e-3  # a key next to a tie of the f16 rounding is a step off: 2^-11 |k|
    assert np.allclose(host(mass)[0], want, rtol=1e-2, atol=0)
    kept = host(p2)[0]
    for g in range(n_kv):
        mg = host(mass)[0, g]
        best = order_of(mg, np.arange(prompt), sinks, prompt - recent)
        assert np.array_equal(kept[g], np.sort(best[:budget]))
    # decode: every step's rows are the kept positions of each head
    now = torch.zeros(1, dtype=torch.int32, device="cuda")
    q1, o1 = torch.empty((1, heads * hd), device="cuda"), torch.empty((1, heads * hd), device="cuda")
    for step in range(6):
        at = prompt + step
        qs, ks, vs = parts(at, at + 1)
        now.fill_(at)
        k1 = rope.apply_dev(ks, now, torch.empty((1, dim), device="cuda"))
        rope.apply_dev(qs, now, q1)
        small.evict_store_dev(0, n_kv, hd, k1, vs, 0, budget, m2[0], p2[0], now, sinks=sinks, recent=recent)
        before = host(m2)[0].astype(np.float64)
        small.attend_mass_dev(0, q1, heads, n_kv, hd, 0, budget - 1, scale, m2[0], o1)
        rows = host(p2)[0]
        for g in range(n_kv):
            assert at in rows[g] and len(set(rows[g])) == budget and set(range(sinks)) <= set(rows[g])
            assert set(range(at - recent + 1, at)) <= set(rows[g])
            hs = slice(g * (heads // n_kv) * hd, (g + 1) * (heads // n_kv) * hd)
            c = slice(g * hd, g * hd + hd)
            o, w, _, _ = attend64(q64[at, hs], k16[:, c], v16[:, c], rows[g], hd, 1, scale)
            assert np.abs(host(o1)[0, hs] - o).max() <= 2e-3
            assert np.allclose(host(m2)[0, g], before[g] + w.sum(0), rtol=1e-2, atol=1e-6)


def test_a_captured_decode_step(hip):
    """Rotation, eviction and weighted attention of a step in one graph, replayed as tokens and positions
    change under it with other work in between: the same bits as the eager calls on a second cache."""
    import torch
    heads, n_kv, hd, budget = 8, 2, 64, 70
    dim = n_kv * hd
    rope = hip.Rope(hd, layout="half")
    sides = []
    for _ in range(2):
        kv, _, _ = make_cache(hip, budget, dim, 950)
        st = {"kv": kv, "mass": cuda(np.abs(normal(951, (n_kv, budget)))), "pos": cuda(np.tile(np.arange(budget, dtype=np.int32), (n_kv, 1))),
              "now": torch.zeros(1, dtype=torch.int32, device="cuda"), "q": torch.zeros((1, heads * hd), device="cuda"),
              "k": torch.zeros((1, dim), device="cuda"), "v": torch.zeros((1, dim), device="cuda"),
              "qr": torch.zeros((1, heads * hd), device="cuda"), "kr": torch.zeros((1, dim), device="cuda"),
              "out": torch.zeros((1, heads * hd), device="cuda"),
              "work": torch.empty(hip.attend_mass_bytes(1, heads, n_kv, hd, budget), dtype=torch.uint8, device="cuda")}
        sides.append(st)

    def step(st):
        rope.apply_dev(st["q"], st["now"], st["qr"])
        rope.apply_dev(st["k"], st["now"], st["kr"])
        st["kv"].evict_store_dev(0, n_kv, hd, st["kr"], st["v"], 0, budget, st["mass"], st["pos"], st["now"], sinks=4, recent=16)
        st["kv"].attend_mass_dev(0, st["qr"], heads, n_kv, hd, 0, budget - 1, hd ** -0.5, st["mass"], st["out"], work=st["work"])

    eager, captured = sides
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        step(captured)
    for i in range(6):
        x = [cuda(normal(960 + 3 * i + j, (1, w))) for j, w in enumerate((heads * hd, dim, dim))]
        for st in sides:
            for name, t in zip(("q", "k", "v"), x):
                st[name].copy_(t)
            st["now"].fill_(budget + i)
        step(eager)
        torch.ones(5000, device="cuda").sum()
        graph.replay()
        for name in ("out", "mass", "pos"):
            assert np.array_equal(host(eager[name]), host(captured[name])), (i, name)
        for a, b in zip(eager["kv"].tensors(0), captured["kv"].tensors(0)):
            assert np.array_equal(host(a), host(b)), i
