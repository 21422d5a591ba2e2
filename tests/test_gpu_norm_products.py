"""The operators around a layer as a program uses them: the norm's codes into BlockLinear's product, and the
norm, router, routing and expert bridges one behind the other."""
import numpy as np
import pytest
import torch

import bridge_case as BC
import layers_case as C
import norm_case as N
import oracle
import routing_case as R
from conftest import gpu_available
from netra_moe import bridges
from netra_moe.linear import BlockLinear
from netra_moe.norm import rms_norm
from netra_moe.routing import route

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.mark.parametrize("T,K,n", [(1, 128, 48), (3, 300, 130), (16, 2048, 2048), (40, 1111, 600), (64, 2048, 8200), (65, 512, 256),
                                   (333, 1000, 700), (1200, 640, 1300), (200, 8000, 300)])
def test_codes_into_the_product(T, K, n):
    """The product of the codes that the norm leaves is that of the values they stand for."""
    g = torch.Generator().manual_seed(T)
    x, res = (torch.randn(T, K, generator=g).to(BF) for _ in range(2))
    w = torch.randn(K, generator=g) * 0.2 + 1.0
    q, s, values = C.weights(n, K, T)
    proj = BlockLinear(q.to(DEV), s.to(DEV))
    r = rms_norm(x.to(DEV), w.to(DEV), residual=res.to(DEV), codes="tiles")
    codes, scale = N.untile(r.codes, r.scale, T, K)
    a = codes * scale.double().repeat_interleave(128, 1)[:, :K]
    N.check_codes(codes, scale, N.norm(N.normalised(x, res), w))
    want, bound = C.product(a, values)
    C.assert_within(proj.forward_codes(r.codes, r.scale, T), want, bound)
    wide = torch.full((T, n + 9), 3.0, dtype=BF, device=DEV)
    proj.forward_codes(r.codes, r.scale, T, wide[:, 5:5 + n])
    C.assert_within(wide[:, 5:5 + n], want, bound)
    assert (wide[:, :5] == 3).all() and (wide[:, 5 + n:] == 3).all()


def test_codes_refusals():
    q, s, _ = C.weights(64, 256, 1)
    proj = BlockLinear(q.to(DEV), s.to(DEV))
    x, w = torch.randn(5, 256, device=DEV), torch.ones(256, device=DEV)
    t, rows = rms_norm(x, w, codes="tiles"), rms_norm(x, w, codes="rows")
    assert proj.forward_codes(t.codes, t.scale, 5).shape == (5, 64)
    for args in [(rows.codes, rows.scale, 5), (t.codes, t.scale, 17), (t.codes.view(torch.float8_e4m3fn), t.scale, 5), (t.codes, t.scale.double(), 5),
                 (t.codes, t.scale, 5, torch.zeros(5, 64, device=DEV)), (t.codes.cpu(), t.scale, 5)]:
        with pytest.raises(ValueError):
            proj.forward_codes(*args)


@pytest.fixture
def model():
    m = BC.build_model()
    for fam in bridges.FAMILIES:
        bridges.check(fam, bridges.load(fam))
    yield m
    torch.cuda.synchronize()
    for fam in bridges.FAMILIES:
        bridges.check(fam, bridges.unload(fam))


def test_norm_and_routing_feed_the_bridges(model):
    """residual + norm -> router bridge -> route -> shared-gate append -> gate/up -> SiLU -> down: the norm's y feeds the
    router, its codes and scales the experts, and the next norm takes the layer's output with the residual."""
    ptr, stream = BC.ptr, BC.stream
    for rows in (1, 16):
        g = torch.Generator().manual_seed(rows)
        x, res = (torch.randn(rows, BC.H, generator=g).to(BF) for _ in range(2))
        w = (torch.randn(BC.H, generator=g) * 0.1 + 1.0).to(BF)
        n = rms_norm(x.to(DEV), w.to(DEV), residual=res.to(DEV), codes="rows")
        logits = torch.empty(rows, BC.E, dtype=BF, device=DEV)
        run = lambda fam, *args: bridges.check("netra_qwen36_" + fam, bridges.launch("netra_qwen36_" + fam, *args, stream()))  # noqa: E731
        run("router_bf16", ptr(logits), ptr(n.y), ptr(model["router_w"]), rows)
        r = route(logits, BC.K)
        ids = torch.empty(rows, BC.KTOT, dtype=torch.int32, device=DEV)
        weights = torch.empty(rows, BC.KTOT, dtype=torch.float32, device=DEV)
        run("shared_gate_append", ptr(ids), ptr(weights), ptr(n.y), ptr(model["shared_w"]), ptr(r.ids), ptr(r.weights), rows)
        gate_up = torch.empty(rows * BC.KTOT, 2 * BC.I, dtype=torch.float32, device=DEV)
        run("moe_gate_up", ptr(n.codes), ptr(n.scale), ptr(model["w13"]), ptr(model["w13_scale"]), ptr(ids), ptr(gate_up), rows)
        h = torch.empty(rows * BC.KTOT, BC.I, dtype=torch.uint8, device=DEV)
        hs = torch.empty(rows * BC.KTOT, BC.I // 128, dtype=torch.float32, device=DEV)
        run("moe_silu_mul_quant", ptr(gate_up), ptr(h), ptr(hs), rows * BC.KTOT)
        out = torch.empty(rows, BC.H, dtype=BF, device=DEV)
        run("moe_down_reduce", ptr(h), ptr(hs), ptr(model["w2"]), ptr(model["w2_scale"]), ptr(weights), ptr(ids), ptr(out), rows)
        after = rms_norm(out, w.to(DEV), residual=n.residual)

        want = N.norm(N.normalised(x, res), w)
        N.check_y(n.y, want)
        N.check_codes(n.codes.cpu().double(), n.scale.cpu(), want)
        chosen = R.choose(logits.cpu(), BC.K)
        assert torch.equal(ids.cpu()[:, :BC.K].long(), chosen) and (ids.cpu()[:, BC.K] == BC.E).all()
        C.assert_within(weights[:, :BC.K].contiguous(), *R.weights(logits, chosen))
        host = model["host"]
        codes, scale = n.codes.cpu().view(torch.uint8).numpy(), n.scale.cpu().numpy()
        ref, _ = oracle.moe_tokens(codes, scale, host["w13"], host["w13_scale"], host["w2"], host["w2_scale"], ids.cpu().numpy(),
                                   weights.cpu().numpy(), np.arange(rows, dtype=np.int64), BC.H, BC.I)
        assert oracle.max_abs_rel(out.cpu().float().numpy(), ref) <= 2e-2
        N.check_y(after.y, N.norm(N.normalised(out.cpu(), n.residual.cpu()), w))
