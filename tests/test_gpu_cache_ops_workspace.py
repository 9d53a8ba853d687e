"""One workspace for a whole run: sized for the most tokens and the longest
ranges, the caller's and the library's own serve every shorter call, captured
ones too.  Tolerances are those of test_gpu_cache_ops.py."""
import numpy as np
import pytest

from conftest import normal
from test_gpu_cache_ops import attend64, cuda, host, make_cache

pytestmark = pytest.mark.gpu

HEADS, N_KV, HD, ROWS = 8, 2, 64, 9000
LENGTHS = [8999, 8193, 8192, 5000, 4097, 2049, 600, 129, 128, 7]


@pytest.fixture(scope="module")
def rows(hip):
    return make_cache(hip, ROWS, N_KV * HD, 3000)


def shared(kv, q, length, out, **kw):
    kv.attend_shared_dev(0, q, HEADS, N_KV, HD, 0, length, None, None, 0, 0.125, out, **kw)


def check(q, k, v, got, length):
    """Each request over the first `length` rows."""
    for i in range(len(q)):
        want, _, u, vm = attend64(q[i], k, v, np.arange(length), HD, N_KV, 0.125)
        assert np.abs(got[i] - want).max() <= u * vm, (i, length)


@pytest.mark.parametrize("n", [2, 5])
def test_one_workspace_for_every_length(hip, rows, n):
    import torch
    kv, k, v = rows
    q, out = normal(3001, (n, HEADS * HD)), torch.empty((n, HEADS * HD), device="cuda")
    work = torch.empty(hip.attend_shared_bytes(n, HEADS, N_KV, HD, LENGTHS[0], 0), dtype=torch.uint8, device="cuda")
    mass_work = torch.empty(hip.attend_mass_bytes(n, HEADS, N_KV, HD, LENGTHS[0]), dtype=torch.uint8, device="cuda")
    for length in LENGTHS:
        print(f"one workspace: {n} over {length}", flush=True)
        shared(kv, cuda(q), length, out, work=work)
        check(q, k, v, host(out), length)
        for m in (n, 1):  # the window's tokens, then a decode step's one
            mass, one = torch.zeros((N_KV, ROWS), device="cuda"), torch.empty((m, HEADS * HD), device="cuda")
            kv.attend_mass_dev(0, cuda(q[:m]), HEADS, N_KV, HD, 0, length - 1, 0.125, mass, one, work=mass_work)
            check(q[m - 1:m], k, v, host(one)[m - 1:], length)
            # m * HEADS softmaxes, to float32 sums of `length` terms
            assert abs(host(mass).sum(dtype=np.float64) - m * HEADS) <= m * HEADS * 1e-4


def test_captured_shorter_calls_need_no_more_scratch(hip, rows):
    """After one call at the longest range on the stream, captures of shorter ones use the library's scratch as it is."""
    import torch
    kv, k, v = rows
    q, out = normal(3002, (5, HEADS * HD)), torch.empty((5, HEADS * HD), device="cuda")
    dq, stream = cuda(q), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        shared(kv, dq, LENGTHS[0], out)
    torch.cuda.synchronize()
    for length in LENGTHS[1:]:
        graph = torch.cuda.CUDAGraph()
        print(f"captured over {length}", flush=True)
        with torch.cuda.graph(graph, stream=stream):
            shared(kv, dq, length, out)
        for _ in range(2):
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            check(q, k, v, host(out), length)
    hip.stream_release(stream.cuda_stream)
