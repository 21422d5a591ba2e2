"""Which kernels the linear layer's rules (csrc/layers/layers_plan.h, compiled for
the host) pick: every kernel form of linear_fp8.hip is reached by the sizes that
layers_forms.py gives the GPU tests, so that a new form, or rules that change,
cannot leave one untested."""
import re
import subprocess
from pathlib import Path

import pytest

import layers_forms as F
from conftest import REPO
from netra_moe import layers, paths

LAYERS = REPO / "netra-kernel_amd" / "csrc" / "layers"


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "plan"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{LAYERS}",
                    str(Path(__file__).with_name("layers_plan_host.cpp")), "-o", str(exe)], check=True)

    def ask(*queries):
        text = "\n".join(" ".join(map(str, q)) for q in queries)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(queries)
        return [[v if v.isalpha() else int(v) for v in line.split()] for line in out]

    return ask


def form(picked, total):
    """A plan's (kernel, splits as layers_forms.py counts them)."""
    *kernel, splits, each = picked
    if splits > 1:
        assert (splits - 1) * each < total < splits * each, "the last split is to be short"
    return (*kernel, min(splits, 2))


@pytest.mark.parametrize("bf16,forms", [(1, F.BF16), (0, F.F32)])
def test_products_reach_the_form_they_are_listed_for(plan, bf16, forms):
    for (want, (rows, ni, nc)), got in zip(forms.items(), plan(*(("product", *s, bf16) for s in forms.values()))):
        assert form(got, -(-nc // 128)) == want, (rows, ni, nc)


def test_weight_gradients_reach_the_form_they_are_listed_for(plan):
    for want, sizes in F.OUTER.items():
        for (rows, n, k), got in zip(sizes, plan(*(("outer", *s) for s in sizes))):
            got[3] //= 64
            assert form(got, -(-rows // 64)) == want, (rows, n, k)


def test_backward_passes_in_one_launch_and_apart(plan):
    for sizes, want in ((F.BACKWARD_IN_ONE, 1), (F.BACKWARD_APART, 0)):
        for (rows, n, k), got in zip(sizes, plan(*(("backward", *s, 1) for s in sizes))):
            assert got == [want], (rows, n, k)
            if want:
                assert plan(("product", rows, k, n, 1))[0][:3] == ["tiles", 128, 64], (rows, n, k)


def test_every_kernel_form_is_listed():
    """The forms that linear_fp8.hip instantiates, by their macros."""
    text = (LAYERS / "linear_fp8.hip").read_text()
    tiles = {tuple(map(int, m)) for m in re.findall(r"^NETRA_PRODUCT_TILE\((\d+), (\d+),", text, re.M)} | {(256, 256)}
    assert "netra_linear_product_256x256_gfx950" in text
    both = {tuple(map(int, m)) for m in re.findall(r"^NETRA_PRODUCTS_FUSED\((\d), (\d)\)", text, re.M)}
    bf16 = {tuple(map(int, m)) for m in re.findall(r"^NETRA_PRODUCT_FUSED\(bf16, uint16_t, (\d), (\d)\)", text, re.M)}
    streams = {tuple(map(int, m)) for m in re.findall(r"^NETRA_PRODUCT_STREAM\((\d), (\d)\)", text, re.M)}
    outer = {tuple(map(int, m)) for m in re.findall(r"^NETRA_OUTER_TILE\((\d+), (\d+),", text, re.M)}
    assert len(tiles) == 5 and both and bf16 and streams and len(outer) == 3
    assert {f[1:3] for f in F.BF16 if f[0] == "fused"} == both | bf16
    assert {f[1:3] for f in F.F32 if f[0] == "fused"} == both
    assert {f[1:3] for f in F.BF16 if f[0] == "stream"} == streams
    assert {f[1:] for f in F.BF16 if f[0] == "tiles"} == {(*t, s) for t in tiles for s in (1, 2)}
    assert set(F.OUTER) == {(*t, s) for t in outer for s in (1, 2)}


def test_quantising_on_the_way_counts_the_workgroups_that_it_launches(plan):
    """33 to 64 rows are quantised on the way by workgroups of one tile of columns, however many
    columns there are: 512 of them are two rounds, 1024 four."""
    for rows, ni, nc in [(64, 8192, 1024), (48, 8192, 2048), (48, 16384, 1024), (40, 8190, 1100), (48, 16384, 128),
                         (64, 32768, 128)]:
        assert plan(("product", rows, ni, nc, 1))[0][:3] == ["stream", 2, 4], (rows, ni, nc)
    for rows, ni, nc in [(48, 4096, 2048), (64, 4096, 1024), (64, 8192, 512), (48, 8192, 128), (64, 12288, 128)]:
        assert plan(("product", rows, ni, nc, 1))[0][:3] == ["fused", 1, 4], (rows, ni, nc)
    for rows, ni, nc in [(20, 8192, 1024), (32, 16384, 1024)]:
        assert plan(("product", rows, ni, nc, 1))[0][:3] == ["fused", 2, 2], (rows, ni, nc)


def test_launches_of_any_size_that_fits_the_memory_fit_their_grids(plan):
    """Threads of a launch's dimension have 32 bits. x, dy, y, dx and dw with the codes and copies
    of a backward pass on fp32 in 288 GB: any sizes up to 2^21."""
    sizes = [1, 17, 65, 333, 1000, 4096, 16384, 1 << 18, (1 << 21) - 1, 1 << 21]
    fit = [(r, n, k) for r in sizes for n in sizes for k in sizes
           if 4 * r * (n + k) + 4 * n * k + 3 * r * n + 2 * r * k < 288e9]
    assert (16384, 1 << 21, 333) in fit and (1, 1 << 21, 16384) in fit
    for size, (prepare, y, dx, dw) in zip(fit, plan(*(("grids", *s) for s in fit))):
        assert 0 < prepare * 256 < 1 << 32 and max(y, dx) * 512 < 1 << 31 and 0 < dw * 512 <= 1 << 31, size


@pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")
@pytest.mark.parametrize("rows,n,k", [(1 << 21, 1 << 21, 128), (1 << 21, 1 << 21, 1 << 21), (128, 1 << 21, 1 << 21)])
def test_more_workgroups_than_a_launch_takes_are_refused_before_any_launch(rows, n, k):
    lib, far = layers.library(), 1 << 44  # addresses that are never followed
    big = 1 << 60
    calls = [("netra_linear_weight_gradient", far, 1, n, 3 * far, 1, k, 5 * far, 0, rows, n, k, 16, big, None),
             ("netra_linear_backward", far, 1, n, 3 * far, 1, k, 16, 16, 5 * far, k, 9 * far, 0, rows, n, k, 16, big, None)]
    if rows > 128:
        calls.append(("netra_linear_forward", far, 1, k, 16, 16, 3 * far, n, rows, n, k, 16, big, None))
    for name, *args in calls:
        assert getattr(lib, name)(*args) == -1, name
        assert "more workgroups" in lib.netra_layers_last_error().decode()
