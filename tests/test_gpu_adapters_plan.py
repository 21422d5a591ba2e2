"""A plan of a batch is refused without its adapters."""
import pytest
import torch

from conftest import gpu_available
from layers_case import weights as fp8_weights
from netra_moe.adapters import make_plan
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
