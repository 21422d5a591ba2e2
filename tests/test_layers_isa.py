"""Static checks of the built libnetra_layers.so (as test_isa_hazards.py and
test_kernel_scratch.py make of the engine's code object): no vector-memory
instruction too close behind a VALU write of a scalar register it reads, no
scratch, no packed fp32, and between a tile kernel's first and last copy into
LDS no other vector-memory operation and only the waits its ring is made for
(a stage's copies times the stages that may stay in flight).

Runs on the CPU; skipped when the library or the ROCm llvm tools are absent."""
import re

import pytest

import test_isa_hazards as I
import test_kernel_scratch as K
from netra_moe import paths

NAME = "libnetra_layers.so"
# kernel -> stages in flight behind a step times a wave's copies per step
RINGS = {"netra_linear_product_256x256_gfx950": 0, "netra_linear_product_256x128_gfx950": 7,
         "netra_linear_product_128x128_gfx950": 10, "netra_linear_product_128x64_gfx950": 8,
         "netra_linear_product_64x64_gfx950": 6, "netra_linear_outer_256x256_gfx950": 0,
         "netra_linear_outer_128x256_gfx950": 6, "netra_linear_outer_128x128_gfx950": 8}


@pytest.fixture
def kernels(monkeypatch):
    monkeypatch.setitem(I.ARTEFACTS, NAME, paths.layers_library())
    return {k: v for k, v in I.disassembly(NAME).items() if k.startswith("netra_")}


def test_no_hazards_and_no_packed_fp32(kernels):
    assert set(RINGS) <= set(kernels) and len(kernels) > 40
    report = {k: h for k, v in kernels.items() if (h := I.hazards(v))}
    assert not report, "\n".join(f"{k}: {h[0]}" for k, h in report.items())
    packed = [k for k, v in kernels.items() if any(re.search(r"\bv_pk_(add|mul|fma)_f32\b", t) for t in v)]
    assert not packed


@pytest.mark.parametrize("kernel", sorted(RINGS))
def test_rings_hold_only_their_copies(kernels, kernel):
    assert not I.ring_violations(kernels[kernel], {0, RINGS[kernel]})


def test_no_scratch(kernels, tmp_path):
    found = {n: b for n, b in K.scratch_bytes(NAME, tmp_path).items() if n.startswith("netra_")}
    assert set(kernels) == set(found) and not {n: b for n, b in found.items() if b}
