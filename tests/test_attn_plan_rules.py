"""How many workgroups attn_plan.h gives a shared range beside own ranges that
are planned as long: all of them where more than two fit a CU, and half where
two do or where a chunk would be one step."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "attn_plan.h"
int main(int, char** v) {
    int a[6];
    for (int i = 0; i < 6; i++) a[i] = std::atoi(v[i + 1]);
    const gllm::SeqPlan p = gllm::seq_plan(a[0], a[1], a[2], a[3], a[4], a[5]);
    std::printf("%d %d\n", a[2] * p.row_blocks * p.chunks, p.chunk);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "t.cpp").write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "gopherllm_amd", "csrc"), str(d / "t.cpp"), "-o", str(d / "t")], check=True)
    return lambda *a: tuple(int(x) for x in subprocess.run([str(d / "t"), *map(str, a)], capture_output=True, text=True, check=True).stdout.split())


@pytest.mark.parametrize("n,heads,n_kv,hd,length", [(33, 40, 8, 80, 32768), (64, 8, 2, 64, 65536), (64, 32, 8, 96, 9973), (17, 32, 8, 32, 32768)])
def test_smaller_heads_keep_all_workgroups(plan, n, heads, n_kv, hd, length):
    alone, _ = plan(n, heads, n_kv, hd, length, 0)
    beside, _ = plan(n, heads, n_kv, hd, length, length // n + 1)
    assert beside == alone > 256


@pytest.mark.parametrize("n,heads,n_kv,hd,length", [(64, 32, 8, 128, 32768), (16, 32, 8, 128, 32768), (64, 32, 8, 120, 4000), (64, 32, 8, 96, 2000)])
def test_two_a_cu_or_single_steps_are_halved(plan, n, heads, n_kv, hd, length):
    alone, chunk = plan(n, heads, n_kv, hd, length, 0)
    beside, _ = plan(n, heads, n_kv, hd, length, length // n + 1)
    assert beside <= 256 < alone and (hd > 96 or chunk == 128)
    short, _ = plan(n, heads, n_kv, hd, length, (length - 1) // n)
    assert short == alone  # own ranges planned shorter than the shared one leave it whole
