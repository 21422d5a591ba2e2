"""Which kernels and grids the rules of the norm, the routing and the adapters
(csrc/layers/layers_plan.h, compiled for the host) pick: what they pick covers the
work, and the GPU tests' sizes reach every kernel."""
import subprocess
from pathlib import Path

import pytest

import test_gpu_adapters
import test_gpu_norm
import test_gpu_operator_calls
from conftest import REPO

LAYERS = REPO / "netra-kernel_amd" / "csrc" / "layers"


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "plan"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{LAYERS}",
                    str(Path(__file__).with_name("operators_plan_host.cpp")), "-o", str(exe)], check=True)

    def ask(queries):
        text = "\n".join(" ".join(map(str, q)) for q in queries)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(queries)
        return [list(map(int, line.split())) for line in out]

    return ask


def test_norm_rows_fit_their_lanes_and_grids(plan):
    sizes = [(T, H) for T in (1, 5, 333, 16384, 1 << 21)
             for H in (1, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384)]
    for (T, H), (waves, chunks, rows, threads, groups, partials) in zip(sizes, plan([("norm", *s) for s in sizes])):
        assert waves * chunks * 512 >= H and threads == 64 * waves * rows
        assert 1 <= groups <= -(-T // rows) and groups * threads < 1 << 32
        assert 1 <= partials <= min(512, -(-T // rows))


def test_norm_sizes_reach_every_kernel(plan):
    got = plan([("norm", *s) for s in test_gpu_norm.SIZES])
    assert {tuple(g[:2]) for g in got} == {(1, 1), (1, 2), (4, 1), (8, 1), (16, 1), (16, 2)}
    # rows that a workgroup loops over
    assert any(g[4] * g[2] < T for g, (T, _) in zip(got, test_gpu_norm.SIZES))
    assert any(g[5] * g[2] < T for g, (T, _) in zip(got, test_gpu_norm.SIZES))


def test_adapters_cover_tokens_contraction_and_columns(plan):
    sizes = [(T, L, r, n, k) for T in (1, 15, 16, 64, 500, 4096, 8191, 8192, 70000, 1 << 21) for L in (1, 7, 128, 1024)
             for r in (1, 16, 17, 64, 128) for n in (1, 512, 2048, 28672) for k in (1, 129, 1111, 8192, 65536)]
    for (T, L, r, n, k), (tile, ranks, tiles, splits, each, wide, fused) in zip(sizes, plan([("adapters", *s) for s in sizes])):
        assert r <= 16 * ranks < max(2 * r, 17)
        parts = min(L + 1, T)  # every one with one token more than whole tiles
        assert tiles >= (T - parts) // tile + parts
        kb = -(-k // 128)
        assert splits * each >= kb > (splits - 1) * each and 1 <= splits <= 16
        assert wide in (1, 2, 4, 8) and (not fused or (tile == 16 and splits == wide == 1))


def test_adapters_sizes_reach_every_kernel(plan):
    got = plan([("adapters", T, L, r, N, K) for T, L, r, K, N, _ in test_gpu_adapters.SIZES])
    assert {(g[0], g[1], g[6]) for g in got} == {(16, r, f) for r in (1, 2, 4, 8) for f in (0, 1)} | {(32, r, 0) for r in (1, 2, 4, 8)}
    assert any(g[3] > 1 for g in got)


def test_adapters_sizes_reach_every_kernel_past_the_caches(plan):
    sizes = test_gpu_operator_calls.ONCE
    once = plan([("once", T, L, r, N) for T, L, r, _, N in sizes])
    got = plan([("adapters", T, L, r, N, K) for T, L, r, K, N in sizes])
    assert all(o == [1] for o in once) and {(g[0], g[1], g[6]) for g in got} == {(t, r, 0) for t in (16, 32) for r in (1, 2, 4, 8)}
    # little B beside as much
    assert plan([("once", 4096, 8, 16, 8192), ("once", 4096, 16, 16, 8192), ("once", 64, 64, 128, 8192)]) == [[0], [1], [0]]


def test_products_of_codes(plan):
    assert plan([("codes", 1, 8191 - 15, 2048), ("codes", 64, 8192, 2048)]) == [[1, 1, 4], [1, 2, 4]]
    assert plan([("codes", 65, 512, 2048)])[0][0] == 2


def test_gradient_groups_loop_past_a_chip(plan):
    assert plan([("select", 1, 16), ("select", 17, 16), ("select", 65536, 16), ("select", 65537, 16), ("select", 1 << 25, 4)]) == \
        [[1], [2], [4096], [4096], [4096]]
