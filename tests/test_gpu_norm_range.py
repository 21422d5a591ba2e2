"""The range of values that include/netra_layers.h states for the norm, at its ends."""
import re

import pytest
import torch

import norm_case as N
from conftest import gpu_available
from layers_case import assert_within
from netra_moe import paths
from netra_moe.norm import rms_norm, rms_norm_gradients

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
DEV = "cuda:0"


def stated():
    text = (paths.REPO_ROOT / "include" / "netra_layers.h").read_text()
    return float(re.search(r"\|r\| below ([0-9e.]+\d)", text).group(1))


@pytest.mark.parametrize("H", [16384, 8192, 1000])
def test_largest_values(H):
    """A row's sum of squares is at most H times the bound's square: 1.6e38 of the fp32 range's 3.4e38."""
    g = torch.Generator().manual_seed(H)
    r = torch.sign(torch.randn(3, H, generator=g)) * (0.99 * stated())
    w, dy = torch.rand(H, generator=g), torch.randn(3, H, generator=g)
    N.check_y(rms_norm(r.to(DEV), w.to(DEV), out_type=torch.float32).y, N.norm(r, w))
    dx, dw = rms_norm_gradients(dy.to(DEV), r.to(DEV), w.to(DEV))
    want, dw_want, bound, dw_bound = N.gradients(dy, r, w, None)
    assert_within(dx, want, bound, "dx")
    assert_within(dw, dw_want, dw_bound, "dw")


@pytest.mark.parametrize("H", [16384, 1000, 1])
def test_smallest_values_without_eps(H):
    """mean(r^2) just above 2^-126. Of squares below it 2^-150 each is lost at most: u of the mean in all."""
    g = torch.Generator().manual_seed(H)
    r = torch.sign(torch.randn(3, H, generator=g)) * (1.05 * 2.0 ** -63)
    w, dy = torch.rand(H, generator=g), torch.randn(3, H, generator=g)
    N.check_y(rms_norm(r.to(DEV), w.to(DEV), eps=0.0, out_type=torch.float32).y, N.norm(r, w, eps=0.0))
    dx, dw = rms_norm_gradients(dy.to(DEV), r.to(DEV), w.to(DEV), eps=0.0)
    want, dw_want, bound, dw_bound = N.gradients(dy, r, w, None, eps=0.0)
    assert_within(dx, want, bound, "dx")
    assert_within(dw, dw_want, dw_bound, "dw")
