"""The operators next to the MoE layer as a training step uses them together: a
block-FP8 projection in front of the layer, the layer's own logits and top-k
ids into counts and balance loss, the loss's gradient back through the router's
weights and the projection, and a gradient step on both weights. Each result
against float64 computed from the same GPU inputs of that stage."""
import numpy as np
import pytest
import torch

import layers_case as C
from conftest import gpu_available
from moe_case import make_inputs
from netra_moe import balance as B
from netra_moe.config import MoEConfig
from netra_moe.layer import MoELayer
from netra_moe.linear import BlockLinear
from test_gpu_balance import check

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DEV = torch.device("cuda", 0)
CASES = [MoEConfig("step_t16", T=16, H=512, E=16, K=2, I=256, S=0, seed=5),
         MoEConfig("step_t40", T=40, H=512, E=24, K=3, I=256, S=1, seed=6),
         MoEConfig("step_t300", T=300, H=1024, E=24, K=3, I=1024, S=1, seed=7)]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: c.name)
def test_projection_layer_loss_and_gradients(cfg):
    K_in = 384
    x0 = C.activations(cfg.T, K_in, seed=cfg.seed).to(DEV)
    q, s, w = C.weights(cfg.H, K_in, seed=cfg.seed)
    proj = BlockLinear(q.to(DEV), s.to(DEV), gradients=True)
    _, moe_weights, _ = make_inputs(cfg, DEV, weights_on_gpu=False)
    moe = MoELayer(cfg, moe_weights, expose=("logits", "topk_ids"), graph=False)

    h = proj.forward(x0)
    C.assert_within(h, *C.product(C.quantised(x0, 1), w), "projection")
    out = moe.forward(h)
    assert torch.isfinite(out.float()).all()
    logits, ids = moe.buffer("logits")[:, :cfg.E], moe.buffer("topk_ids")
    want = C.counts(ids, cfg.E)
    assert want.sum() == cfg.T * cfg.K  # the shared expert's slot is not counted
    np.testing.assert_array_equal(B.expert_counts(ids, cfg.E).cpu().numpy(), want)
    r = B.balance_loss(logits, ids, bias=moe_weights["router_bias"], coefficient=0.01)
    np.testing.assert_array_equal(r.counts.cpu().numpy(), want)
    check(r, logits, want, 0.01, bias=moe_weights["router_bias"].cpu())

    # through the router (bf16 weights, plain torch) and the projection
    dh = (r.grad.float() @ moe_weights["router_w"][:cfg.E].float()).to(torch.bfloat16)
    dx, dw = proj.backward(dh, x0)
    C.assert_within(dx, *C.product(C.quantised(dh, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dh, x0), "dw")
    # a second micro-batch adds to dw
    both = proj.weight_gradient(dh, x0, dw.clone(), accumulate=True)
    assert torch.equal(both, dw + dw)

    # the step's new weights make a layer of their own
    new = BlockLinear.from_float(w.float().to(DEV) - 0.1 * dw, gradients=True)
    assert new.forward(x0).shape == (cfg.T, cfg.H)
    moe.close()


def test_decode_steps_accumulate_the_expert_load():
    cfg = MoEConfig("load_t1", T=1, H=512, E=16, K=2, I=256, S=0, seed=8)
    _, moe_weights, _ = make_inputs(cfg, DEV, weights_on_gpu=False)
    moe = MoELayer(cfg, moe_weights, expose=("topk_ids",), graph=False)
    q, s, _ = C.weights(cfg.H, 256, seed=9)
    proj = BlockLinear(q.to(DEV), s.to(DEV))
    load, want = torch.zeros(cfg.E, dtype=torch.int32, device=DEV), np.zeros(cfg.E, dtype=np.int64)
    for i in range(12):
        moe.forward(proj.forward(C.activations(1, 256, seed=i).to(DEV)))
        B.expert_counts(moe.buffer("topk_ids"), cfg.E, out=load, accumulate=True)
        want += C.counts(moe.buffer("topk_ids"), cfg.E)
    np.testing.assert_array_equal(load.cpu().numpy(), want)
    assert want.sum() == 24
    moe.close()
