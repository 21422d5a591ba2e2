"""Balance loss of more tokens than the workgroups take in one pass (16384 of up to
256 experts, 4096 of more), counted by workgroups of 1024 threads from 16385 tokens
on: against the float64 formulas within the bounds of test_gpu_balance.py."""
import numpy as np
import pytest
import torch

import layers_case as C
from test_gpu_balance import BF16, DEV, F32, check, pytestmark, routing  # noqa: F401
from netra_moe import balance as B


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,E,K,extra", [(16385, 40, 2, 1), (20003, 128, 4, 0), (33001, 255, 8, 1), (40001, 16, 3, 0),
                                         (4097, 300, 6, 0), (9001, 513, 3, 1), (16500, 1024, 2, 0), (70001, 3, 1, 0)])
def test_balance_over_several_passes(T, E, K, extra, masked, dt):
    logits, ids = routing(T, E, K, seed=T + E, extra=extra, dtype=dt)
    mask = None
    if masked:
        mask = torch.rand(T, generator=torch.Generator().manual_seed(2)) < 0.7
        logits[~mask] = torch.nan
        ids[~mask] = 123456
    z, m = logits.to(DEV)[:, :E], None if mask is None else mask.to(DEV)
    r = B.balance_loss(z, ids.to(DEV), mask=m, coefficient=0.3)
    want = C.counts(ids, E, mask)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), want)
    check(r, logits[:, :E], want, 0.3, mask=mask)
    given = B.balance_loss(z, counts=r.counts, mask=m, coefficient=0.3)
    assert torch.equal(given.loss, r.loss) and torch.equal(given.grad, r.grad)
    again = B.balance_loss(z, ids.to(DEV), mask=m, coefficient=0.3)
    assert torch.equal(again.loss, r.loss) and torch.equal(again.grad, r.grad)
