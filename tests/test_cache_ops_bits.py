"""What the two f16 parts of a query and of a weight are worth, by emulation in
numpy: the tolerances of test_gpu_cache_ops_bits.py hold with both, and tell
when one is missing or the weights' second part is cut."""
import numpy as np
import pytest

from conftest import normal
from test_gpu_cache_ops_bits import TOL, TOL_HEAVY

LIFT = 8  # the largest weight is 2^LIFT at least


def parts(x, second=True, cut=False):
    """x as the sum of two f16 values, the second to nearest or cut towards zero."""
    hi = x.astype(np.float16).astype(np.float64)
    if cut:
        step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-300))) - 10, -24))
        hi = np.trunc(x / step) * step
    rest = x - hi
    if not second:
        return hi
    if not cut:
        return hi + rest.astype(np.float16).astype(np.float64)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(rest), 1e-300))) - 10, -24))
    return hi + np.trunc(rest / step) * step


def attend(q, k, v, scale, q_second=True, w_second=True, cut=False):
    top = np.exp2(14 - np.floor(np.log2(np.abs(q).max(-1, keepdims=True))))
    s = parts(q * top, q_second) / top @ k.T * scale
    w = np.exp(s - s.max(-1, keepdims=True)) * 2.0 ** LIFT
    return parts(w, w_second, cut) @ v / w.sum(-1, keepdims=True)


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("rows,hd,length", [(16, 128, 130), (25, 80, 257), (45, 40, 1000), (132, 128, 700), (64, 128, 4001)])
def test_both_parts_are_needed(rows, hd, length):
    q, k, v = (normal(i, s).astype(np.float64) for i, s in enumerate([(rows, hd), (length, hd), (length, hd)]))
    k, v = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
    s = q @ k.T * hd ** -0.5
    w = np.exp(s - s.max(-1, keepdims=True))
    want = w @ v / w.sum(-1, keepdims=True)
    assert off(attend(q, k, v, hd ** -0.5), want) <= TOL / 4
    assert off(attend(q, k, v, hd ** -0.5, q_second=False), want) >= 10 * TOL
    assert off(attend(q, k, v, hd ** -0.5, w_second=False), want) >= 10 * TOL


@pytest.mark.parametrize("length", [3000, 30000])
def test_small_weights_beside_heavy_rows_are_rounded_to_nearest(length):
    hd, rows = 32, 8
    scale, heavy = hd ** -0.5, np.arange(length) % 32 == 5
    k, v, q = normal(1, (length, hd), 0.5).astype(np.float64), 1 + normal(2, (length, hd), 0.1).astype(np.float64), normal(3, (rows, hd))
    k[heavy], v[heavy] = 0, 0
    k[:, 0] = np.where(heavy, 8, 0)
    k, v, q = (x.astype(np.float16).astype(np.float64) if x is not q else q.astype(np.float64) for x in (k, v, q))
    q[:, 0] = 18 * np.log(2) / (8 * scale)
    s = q @ k.T * scale
    w = np.exp(s - s.max(-1, keepdims=True))
    want = w @ v / w.sum(-1, keepdims=True)
    assert off(attend(q, k, v, scale), want) <= TOL_HEAVY / 4
    assert off(attend(q, k, v, scale, cut=True), want) >= 2 * TOL_HEAVY
