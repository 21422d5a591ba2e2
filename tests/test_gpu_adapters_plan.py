"""A plan of a batch: refused without its adapters, and of the longest batches."""
import pytest
import torch

import adapters_case as C
from conftest import gpu_available
from layers_case import assert_within
from layers_case import weights as fp8_weights
from netra_moe.adapters import LowRankAdapters, make_plan
from netra_moe.linear import BlockLinear

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF = torch.bfloat16
DEV = "cuda:0"


def test_a_projection_refuses_a_plan_without_its_adapters():
    q, s, _ = fp8_weights(48, 64, 1)
    proj = BlockLinear(q.to(DEV), s.to(DEV))
    x = torch.randn(5, 64, device=DEV).to(BF)
    plan = make_plan(torch.zeros(5, dtype=torch.int32, device=DEV), 2)
    out = torch.zeros(5, 48, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="plan"):
        proj.forward(x, out, plan=plan)
    assert not out.any()
    assert proj.forward(x, out) is out and out.any()


@pytest.mark.parametrize("T,L", [(1 << 21, 1), (1 << 21, 1024), ((1 << 21) - 77, 40), (300001, 3)])
def test_longest_batches(T, L):
    r, K, N = 3, 8, 5
    a, b, s = (v.to(DEV) for v in C.adapters(L, r, K, N, L))
    lora = LowRankAdapters(a, b, s)
    g = torch.Generator(device=DEV).manual_seed(T)
    x, y = (torch.randn(T, n, generator=g, device=DEV).to(BF) for n in (K, N))
    ids = torch.randint(0 if L == 1 else -1, L, (T,), generator=g, device=DEV, dtype=torch.int32)
    got = lora.add(y, x, lora.plan(ids))
    none, at = (ids < 0)[:, None], ids.clamp_min(0).long()
    want, bound = y.double(), torch.zeros(T, N, dtype=torch.float64, device=DEV)
    a, b, s = a.double(), b.double(), s.double()
    for j in range(r):  # (the bound of adapters_case.py, a rank at a time)
        terms = x.double() * a[at, j]
        u, size = terms.sum(1) * s[at], terms.abs().sum(1) * s[at]
        part = torch.where(none, 0.0, u[:, None] * b[at, :, j])
        want += part
        bound += torch.where(none, 0.0, ((K + 41) * C.U * size + 2.0 ** -16 * u.abs())[:, None] * b[at, :, j].abs() + (4 * r + 16) * C.U * part.abs())
    bound += torch.where(none, 0.0, 2 * C.U * (y.double().abs() + want.abs()))
    assert_within(got, want.cpu(), bound.cpu())
    assert torch.equal(got[ids < 0], y[ids < 0])
