"""Accumulated attention weights where scores are far from zero, of any sign or
all alike, against the definition in 64 bits (the tolerances are those of
test_gpu_cache_ops.py, whose score bound S counts the offset); a cache's rows as
tensors; and batches with padding."""
import numpy as np
import pytest

from conftest import normal
from test_gpu_cache_ops import NAN, attend64, cuda, host, make_cache

pytestmark = pytest.mark.gpu


def check_mass(hip, n, heads, n_kv, hd, start, end, seed, offset=0.0, std=1.0, scale=None):
    """attend_mass_dev with every score moved by `offset` through a constant channel of the keys."""
    import torch
    rows, scale = end + 2, hd ** -0.5 if scale is None else scale
    kv, k, v = make_cache(hip, rows, n_kv * hd, seed, std=std)
    q = normal(seed + 5, (n, heads * hd))
    if offset:
        k[:, ::hd] = 16.0
        q[:, ::hd] = offset / (16.0 * scale)
        kv.tensors(0)[0].copy_(cuda(k.astype(np.float16)))
    before = np.abs(normal(seed + 6, (n_kv, rows)))
    mass, out = cuda(before), torch.full((n, heads * hd), NAN, device="cuda")
    print(f"mass n {n} heads {heads}/{n_kv}x{hd} rows {start}..{end} offset {offset} std {std} scale {scale}", flush=True)
    kv.attend_mass_dev(0, cuda(q), heads, n_kv, hd, start, end, scale, mass, out)
    got, got_mass = host(out), host(mass)
    want_mass, slack = before.astype(np.float64), np.zeros((n_kv, rows))
    for i in range(n):
        at = np.arange(start, end - (n - 1) + i + 1)
        want, w, u, vm = attend64(q[i], k, v, at, hd, n_kv, scale)
        assert np.abs(got[i] - want).max() <= u * vm, i
        per = w.reshape(n_kv, heads // n_kv, -1).sum(1)
        want_mass[:, at] += per
        slack[:, at] += u * per
    # and the roundings of n * r additions and of the one onto what was there
    slack += (n * heads // n_kv + 2) * 2.0 ** -24 * want_mass
    assert np.isfinite(got_mass).all()
    assert (np.abs(got_mass - want_mass) <= slack + 1e-30).all()


# one token of up to 16 heads a kv head keeps its scores; the others make them again, most in part-filled tiles of 16 rows
SHAPES = [(1, 8, 2, 64, 0, 300), (1, 15, 1, 128, 3, 70), (3, 12, 3, 128, 0, 200), (7, 10, 2, 80, 2, 301), (33, 4, 2, 32, 0, 90),
          (2, 8, 1, 96, 0, 40), (1, 71, 1, 64, 0, 130), (5, 32, 8, 128, 0, 33)]


@pytest.mark.parametrize("offset", [-150.0, 150.0, -1000.0])
@pytest.mark.parametrize("n,heads,n_kv,hd,start,end", SHAPES)
def test_mass_of_scores_far_from_zero(hip, n, heads, n_kv, hd, start, end, offset):
    """A constant channel of the keys moves every score alike, which softmax does not see."""
    check_mass(hip, n, heads, n_kv, hd, start, end, 1000 + n + hd, offset=offset)


@pytest.mark.parametrize("std,scale", [(30.0, None), (1.0, -0.3), (1.0, 0.0), (6e-8, 1e4), (1.0, 4.0)])
@pytest.mark.parametrize("n,heads,n_kv,hd,start,end", SHAPES)
def test_mass_score_ranges(hip, n, heads, n_kv, hd, start, end, std, scale):
    """Scores from all equal to one row that takes it all, and keys from f16's least subnormals to large ones."""
    check_mass(hip, n, heads, n_kv, hd, start, end, 1100 + n + hd, std=std, scale=scale)


def test_tensors_are_the_caches_rows(hip):
    """Not copies: the addresses are the cache's, and what is written through them is read back from it."""
    import torch
    kv = hip.KVCacheF16(2, 24, 40, 9)
    for l in range(2):
        k, v = kv.tensors(l)
        assert (k.data_ptr(), v.data_ptr()) == (kv.k_ptr(l), kv.v_ptr(l)) and k.get_device() == v.get_device() == torch.cuda.current_device()
        k.fill_(1.5 + l)
        v.fill_(-2.0 - l)
        torch.cuda.synchronize()
        rk, rv = kv.read(l, 0, 9)
        assert (rk.view(np.float16) == 1.5 + l).all() and (rv.view(np.float16) == -2.0 - l).all()


@pytest.mark.parametrize("n,heads,n_kv,hd,length", [(3, 8, 2, 64, 200), (9, 40, 8, 80, 257), (33, 32, 8, 128, 700), (70, 32, 8, 128, 129)])
@pytest.mark.parametrize("pad", [NAN, float("inf"), -float("inf"), 3e38])
def test_shared_padded_batch(hip, n, heads, n_kv, hd, length, pad):
    """What stands in the queries of a batch's padding, and rows of `out` behind the batch, concern nobody."""
    import torch
    kv, _, _ = make_cache(hip, length + 5 * n, n_kv * hd, 1200)
    live = np.arange(n) % 3 != 1
    lens = cuda(np.where(live, 1 + np.arange(n) % 5, 0).astype(np.int32))
    starts = cuda((length + 5 * np.arange(n)).astype(np.int32))
    q = normal(1201, (n, heads * hd))
    outs = []
    print(f"padded batch: {n} of {heads}/{n_kv}x{hd}, {pad}", flush=True)
    for fill in (0.0, pad):
        q[~live] = fill
        out = torch.full((n + 2, heads * hd), 7.0, device="cuda")
        kv.attend_shared_dev(0, cuda(q), heads, n_kv, hd, 0, length, starts, lens, 5, hd ** -0.5, out)
        outs.append(host(out))
    assert np.isfinite(outs[0]).all()
    assert np.array_equal(outs[0][:n][live], outs[1][:n][live]) and (outs[1][n:] == 7.0).all()


@pytest.mark.parametrize("layout,rot", [("half", 64), ("interleaved", 64), ("half", 20), ("interleaved", 22)])
def test_rope_padded_batch(hip, layout, rot):
    """Padding (row -1) of NaN at any position stores nothing and leaves the others as they are without it."""
    rope, n, hd = hip.Rope(64, rot_dim=rot, layout=layout), 9, 64
    live = np.arange(n) % 3 != 1
    q, k, v = (normal(1210 + i, (n, 2 * hd)) for i in range(3))
    pos, rows = np.arange(n, dtype=np.int32) * 1000, np.where(live, np.arange(n), -1).astype(np.int32)
    got = []
    for keep in (np.ones(n, bool), live):
        kv = hip.KVCacheF16(1, 2 * hd, 2 * hd, n + 1)
        a, b, c = (x.copy() for x in (q, k, v))
        for x in (a, b, c):
            x[~keep] = NAN
        p = np.where(keep, pos, -(2**31)).astype(np.int32)
        dq = cuda(a)
        kv.store_rope_dev(0, rope, dq, cuda(b), cuda(c), cuda(p), cuda(rows))
        got.append((host(dq)[live], *(host(t) for t in kv.tensors(0))))
    for x, y in zip(*got):
        assert np.array_equal(x, y)
    for t in got[1][1:]:
        assert (t[np.r_[~live, True]] == 0).all() and (t[np.r_[live, False]] != 0).any()
