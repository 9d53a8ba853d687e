"""Accumulated attention weights where scores are far from zero, of any sign or
all alike, against the definition in 64 bits; the tolerances are those of
test_gpu_cache_ops.py, whose score bound S counts the offset."""
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
