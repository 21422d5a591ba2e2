"""Static check of the kernel that runs both products of a small backward pass
(netra_linear_backward_small_gfx950): it holds two rings of copies, one per branch,
and each has to be what test_layers_isa.py asks of a kernel with one. The rings wait
for 6 (dx: two steps of three copies) and 8 (dw: two of four) copies in flight; the
first full wait is behind the first ring, so what follows it is the second's.

Runs on the CPU; skipped when the library or the ROCm llvm tools are absent."""
import re

import pytest

import test_isa_hazards as I
from netra_moe import paths

NAME = "libnetra_layers.so"
DX, DW = (6, 4 * 3), (8, 4 * 4)  # copies in flight behind a step, copy instructions: four stages each
_COPY = re.compile(r"buffer_load_dword\w*\s.*\blds\b")


def rings(lines):
    """The instructions up to the second ring's first copy, and the rest."""
    text = [t.split("//")[0].strip() for t in lines]
    first = next(i for i, t in enumerate(text) if _COPY.match(t))
    drain = next(i for i in range(first, len(text)) if re.match(r"s_waitcnt.*vmcnt\(0\)", text[i]))
    second = next(i for i in range(drain, len(text)) if _COPY.match(text[i]))
    return text[:second], text[second:]


def check(lines):
    parts = [(sum(bool(_COPY.match(t)) for t in part), part) for part in rings(lines)]
    bad = []
    for (copies, part), (waits, expected) in zip(parts, (DX, DW)):
        if copies != expected:
            bad.append(f"{copies} copies in a ring that has {expected}")
        bad += I.ring_violations(part, {0, waits})
        if not any(f"vmcnt({waits})" in t for t in part):
            bad.append(f"no wait for {waits}")
    return bad


@pytest.fixture
def lines(monkeypatch):
    monkeypatch.setitem(I.ARTEFACTS, NAME, paths.layers_library())
    return I.disassembly(NAME)["netra_linear_backward_small_gfx950"]


def test_both_rings_hold_only_their_copies(lines):
    assert not check(lines)


def test_the_check_sees_a_foreign_operation_in_either_ring(lines):
    text = [t.split("//")[0].strip() for t in lines]
    copies = [i for i, t in enumerate(text) if _COPY.match(t)]
    for ring in (copies[:DX[1]], copies[DX[1]:]):
        at = ring[len(ring) // 2] + 1
        for foreign in ("global_load_dword v5, v[6:7], off", "s_waitcnt vmcnt(3)",
                        "buffer_load_dword v2, s[4:7], s1 offen lds"):
            assert check(text[:at] + [foreign] + text[at:]), foreign
