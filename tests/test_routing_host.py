"""The routing without a GPU: refusals (before any launch) and the 64-bit forms against autograd."""
import ctypes

import pytest
import torch

import routing_case as R
from netra_moe import layers, paths, routing
from test_layers_host import A, B, D, refused

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")
F = ctypes.c_float


@pytest.mark.parametrize("change", [
    dict(z=0), dict(z=A + 1), dict(zt=2), dict(zs=31), dict(zs=1 << 27), dict(bias=D + 1), dict(T=(1 << 25) + 1), dict(T=1 << 31), dict(E=0), dict(E=1025, zs=2000),
    dict(k=0), dict(k=17), dict(k=33), dict(shared=2), dict(shared=1, k=16, zs=40, s=20), dict(shared=1), dict(scoring=2), dict(G=0),
    dict(G=3), dict(G=17, E=34, zs=40), dict(G=4, top=0), dict(G=4, top=5), dict(G=4, top=1, k=9, s=9), dict(score=2),
    dict(G=16, E=16, top=16, score=1), dict(scale=float("nan")), dict(ids=0), dict(ids=B + 2), dict(s=7), dict(w=0), dict(w=D + 2),
    dict(ids=A), dict(w=A + 64), dict(w=B + 4), dict(ids=3 * A + 8, bias=3 * A), dict(w=5 * A, mask=5 * A + 16)])
def test_select_refusals(change):
    a = dict(z=A, zt=0, zs=32, bias=None, mask=None, T=50, E=32, k=8, shared=0, scoring=0, G=1, top=1, score=0, renorm=1,
             scale=1.0, ids=B, s=8, w=D)
    a.update(change)
    refused("netra_router_select", a["z"], a["zt"], a["zs"], a["bias"], a["mask"], a["T"], a["E"], a["k"], a["shared"],
            a["scoring"], a["G"], a["top"], a["score"], a["renorm"], F(a["scale"]), a["ids"], a["s"], a["w"], a["s"], None)


@pytest.mark.parametrize("change", [
    dict(dw=0), dict(dw=A + 2), dict(ds=7), dict(z=0), dict(z=B + 1), dict(zt=2), dict(zs=31), dict(zs=1 << 27), dict(ids=0),
    dict(ids=D + 1), dict(s=7), dict(T=1 << 31), dict(E=0), dict(k=0), dict(k=17, ds=20, s=20), dict(shared=2), dict(scoring=2),
    dict(scale=float("nan")), dict(g=0), dict(g=4 * A + 1), dict(gs=31), dict(gs=1 << 27), dict(g=B), dict(g=A + 32), dict(g=D + 4),
    dict(shared=1)])
def test_gradient_refusals(change):
    a = dict(dw=A, ds=8, z=B, zt=0, zs=32, ids=D, s=8, T=50, E=32, k=8, shared=0, scoring=0, renorm=1, scale=1.0, g=4 * A, gs=32)
    a.update(change)
    refused("netra_router_select_gradient", a["dw"], a["ds"], a["z"], a["zt"], a["zs"], a["ids"], a["s"], None, a["T"], a["E"],
            a["k"], a["shared"], a["scoring"], a["renorm"], F(a["scale"]), a["g"], a["gs"], 0, None)


def test_no_tokens_launch_nothing():
    lib = layers.library()
    assert lib.netra_router_select(None, 0, 0, None, None, 0, 8, 2, 0, 0, 1, 1, 0, 1, F(1), None, 0, None, 0, None) == 0
    assert lib.netra_router_select_gradient(None, 0, None, 0, 0, None, 0, None, 0, 8, 2, 0, 0, 1, F(1), None, 0, 0, None) == 0


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU tensor"):
        routing.route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError, match="GPU tensor"):
        routing.route_gradient(torch.zeros(2, 2), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("shared", [False, True])
def test_gradient_formula_against_autograd_and_differences(scoring, renormalise, shared):
    z = R.inputs(7, 11, 3, torch.float32, shared).double().requires_grad_()
    ids = R.choose(z[:, :11].detach(), 3)
    dw = torch.randn(7, 3 + shared, generator=torch.Generator().manual_seed(1), dtype=torch.float64)

    def w(z):
        x = z[:, :11]
        s = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, 1)
        s = s.gather(1, ids)
        s = 2.5 * (s / s.sum(1, keepdim=True) if renormalise else s)
        return torch.cat([s, torch.sigmoid(z[:, 11:])], 1) if shared else s

    want, = torch.autograd.grad((w(z) * dw).sum(), z)
    got, bound = R.gradient(dw, z.detach(), ids, scoring, renormalise, 2.5, shared)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-15)
    assert torch.autograd.gradcheck(w, (z,))
    value, _ = R.weights(z.detach(), ids, scoring, renormalise, 2.5, shared)
    assert torch.allclose(value, w(z.detach()), rtol=1e-13)
    # the bounds see a wrong scale of a hundred thousandth
    with pytest.raises(AssertionError):
        R.assert_within((got * 1.0001).float(), got, bound)


def test_choice_of_groups_by_hand():
    z = torch.tensor([[1.0, 2.0, 5.0, 0.0, 3.0, 3.0, -1.0, 4.0]])
    assert R.choose(z, 2, groups=4, top_groups=2).tolist() == [[2, 7]]
    # sums of two: 3, 5, 6, 3 of the logits' sigmoids keep their order here
    assert R.choose(z, 3, "sigmoid", groups=4, top_groups=2, group_score="top2").tolist() == [[4, 5, 1]]
    assert R.choose(z, 2, "sigmoid", bias=torch.tensor([9.0, 0, 0, 0, 0, 0, 9.0, 0])).tolist() == [[0, 6]]
    assert R.choose(torch.zeros(1, 6), 3).tolist() == [[0, 1, 2]]
