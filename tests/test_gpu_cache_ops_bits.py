"""How many bits attention over cache ranges carries: errors in the 2-norm over
all outputs, against 64 bits on the device.

N(0, 1) inputs at scale hd^-0.5, relative to the outputs (TOL).  Roundings are
independent, so they add in squares; each is half a step at most, 0.58 of that
in the mean square.  In units of 2^-24: a score's sum of up to 2 hd = 256
products, partial sums on their way to a score of size 1: 16 * 0.58 * 0.7 = 6.5;
q's second part 1.2; the score times the scale, less the base (8 bits and more
before the largest): 8 * 0.58 * ln 2 = 3.2; the exponential 2; the weight's
second part 4 * 0.58 = 2.3; the sums of up to 500 products of weights and
values, and of the weights: 22 * 0.58 * 0.7 = 9 each.  The root of the squares'
sum is 15, 9e-7; 2e-6 is a little over twice that.  Without either second part
the error is 1e-4 (test_cache_ops_bits.py).

A heavy row of weight 2^18 (and none of the values) in each 32 rows (TOL_HEAVY):
the others' weights stay 2^-18 of the largest, and their sum is the whole
output.  Relative to it: the heavy score 18 ln 2 = 12.5 times the two parts of q
(2), scale * log2(e) (1.5), one sum (1) and its scaling (1), 5.5 * 2^-24 in all
when they add up: 4.1e-6; the sums as above 1e-6; and the light weights' second
part, which ends 2^-33 below the largest weight, 2^-15 relative to each:
0.58 * 2^-15 / sqrt(rows) when it is to nearest, 3e-7 for 3000 rows, but
2^-15 = 3e-5 on one side when it is cut.  8e-6 lies between.
"""
import numpy as np
import pytest

from conftest import normal
from test_gpu_cache_ops import cuda, make_cache

pytestmark = pytest.mark.gpu

TOL, TOL_HEAVY = 2e-6, 8e-6


def outputs64(q, k, v, heads, n_kv, hd, scale, spans):
    """q (n, heads * hd), k and v (rows, dim) on the device; spans: the row indices of each request, or one range for all."""
    import torch
    n, r = q.shape[0], heads // n_kv
    out = torch.zeros((n, n_kv, r, hd), dtype=torch.float64, device="cuda")
    q64 = q.double().view(n, n_kv, r, hd)
    for g in range(n_kv):
        kg, vg = (x[:, g * hd:g * hd + hd].double() for x in (k, v))
        if isinstance(spans, slice):
            w = torch.softmax(q64[:, g].reshape(n * r, hd) @ kg[spans].T.contiguous() * scale, -1)
            out[:, g] = (w @ vg[spans]).view(n, r, hd)
        else:
            for i, at in enumerate(spans):
                w = torch.softmax(q64[i, g] @ kg[at].T.contiguous() * scale, -1)
                out[i, g] = w @ vg[at]
    return out.view(n, -1)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("n,heads,n_kv,hd,length,most", [
    (1, 32, 8, 128, 1000, 0), (3, 32, 8, 128, 130, 40), (5, 40, 8, 80, 257, 60), (9, 10, 2, 40, 1000, 32), (17, 32, 8, 128, 515, 17),
    (33, 32, 8, 128, 700, 7), (12, 32, 8, 128, 0, 900),
    # 32 rows a wave
    (1024, 8, 1, 128, 4001, 0), (2048, 8, 1, 80, 3201, 0), (2048, 8, 1, 40, 6503, 0), (63, 65, 1, 128, 7815, 0)])
def test_shared_bits(hip, n, heads, n_kv, hd, length, most):
    import torch
    rows = length + n * most + 1
    kv, _, _ = make_cache(hip, rows, n_kv * hd, 2000 + hd)
    q, scale = cuda(normal(2001, (n, heads * hd))), float(np.float32(hd ** -0.5))
    out = torch.empty((n, heads * hd), device="cuda")
    starts = cuda((length + most * np.arange(n)).astype(np.int32))
    lens = cuda(np.full(n, most, np.int32))
    print(f"shared, bits: {n} of {heads}/{n_kv}x{hd} over {length} + {most}", flush=True)
    kv.attend_shared_dev(0, q, heads, n_kv, hd, 0, length, starts if most else None, lens if most else None, most, scale, out)
    spans = slice(0, length) if most == 0 else \
        [torch.cat([torch.arange(length), length + most * i + torch.arange(most)]).cuda() for i in range(n)]
    assert off(out, outputs64(q, *kv.tensors(0), heads, n_kv, hd, scale, spans)) <= TOL


@pytest.mark.parametrize("n,heads,n_kv,hd,rows", [(1, 32, 8, 128, 900), (40, 8, 2, 128, 700), (1024, 8, 1, 128, 5200)])
def test_mass_bits(hip, n, heads, n_kv, hd, rows):
    """What every token sees of the keys, and each row's weight from all tokens."""
    import torch
    kv, _, _ = make_cache(hip, rows, n_kv * hd, 2010)
    q, scale, r = cuda(normal(2011, (n, heads * hd))), float(np.float32(hd ** -0.5)), heads // n_kv
    out, mass = torch.empty((n, heads * hd), device="cuda"), torch.zeros((n_kv, rows), device="cuda")
    print(f"mass, bits: {n} of {heads}/{n_kv}x{hd} over {rows}", flush=True)
    kv.attend_mass_dev(0, q, heads, n_kv, hd, 0, rows - 1, scale, mass, out)
    k, v = kv.tensors(0)
    seen = torch.arange(rows, device="cuda") <= rows - n + torch.arange(n, device="cuda")[:, None]
    want, per = torch.zeros((n, n_kv, r, hd), dtype=torch.float64, device="cuda"), torch.zeros((n_kv, rows), dtype=torch.float64, device="cuda")
    for g in range(n_kv):
        c = slice(g * hd, g * hd + hd)
        s = (q.double().view(n, n_kv, r, hd)[:, g].reshape(n * r, hd) @ k[:, c].double().T.contiguous()).view(n, r, rows) * scale
        w = torch.softmax(s.masked_fill(~seen[:, None], -np.inf), -1)
        want[:, g], per[g] = (w.view(n * r, rows) @ v[:, c].double()).view(n, r, hd), w.sum((0, 1))
    assert off(out, want.view(n, -1)) <= TOL
    assert off(mass, per) <= TOL


@pytest.mark.parametrize("n,heads,n_kv,hd,length", [
    (1, 8, 1, 64, 40000),       # waves take positions
    (40, 8, 2, 128, 30000),     # waves take rows
    (4096, 8, 1, 32, 3000),     # one workgroup a block of rows takes the whole range
    (8192, 8, 1, 32, 3000)])    # and 32 rows a wave
def test_shared_small_weights_beside_heavy_rows(hip, n, heads, n_kv, hd, length):
    import torch
    kv = hip.KVCacheF16(1, n_kv * hd, n_kv * hd, length)
    scale, heavy = float(np.float32(hd ** -0.5)), np.arange(length) % 32 == 5
    k, v = normal(2020, (length, n_kv * hd), 0.5), 1 + normal(2021, (length, n_kv * hd), 0.1)
    k[heavy], v[heavy] = 0, 0
    k[:, ::hd] = np.where(heavy, 8, 0)[:, None]
    tk, tv = kv.tensors(0)
    tk.copy_(cuda(k.astype(np.float16)))
    tv.copy_(cuda(v.astype(np.float16)))
    q = normal(2022, (n, heads * hd))
    q[:, ::hd] = 18 * np.log(2) / (8 * scale) + q[:, ::hd] / 64
    q, out = cuda(q), torch.empty((n, heads * hd), device="cuda")
    print(f"shared, heavy rows: {n} of {heads}/{n_kv}x{hd} over {length}", flush=True)
    kv.attend_shared_dev(0, q, heads, n_kv, hd, 0, length, None, None, 0, scale, out)
    err = off(out, outputs64(q, tk, tv, heads, n_kv, hd, scale, slice(0, length)))
    print("off by", err, flush=True)
    assert err <= TOL_HEAVY
