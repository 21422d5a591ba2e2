"""netra_moe.routing where the kept groups hold hardly more experts than are chosen, where biases and
logits are infinite or NaN, and where gradients of small scores are large (forms and bounds of routing_case.py)."""
import pytest
import torch

import routing_case as R
from conftest import gpu_available
from layers_case import assert_within
from netra_moe.routing import route, route_gradient
from test_gpu_routing import check_route

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = "cuda:0"


def near_pairs(T, E, seed, every):
    """fp32 logits; in each `every`-th token every expert has a neighbour that is one or two roundings away."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(T, E, generator=g) * 1.5
    half = E // 2
    for t in range(0, T, every):
        order = torch.randperm(E, generator=g)
        z[t, order[half:2 * half]] = z[t, order[:half]] * (1 + 2.0 ** -23 * torch.randint(0, 3, (half,), generator=g))
    return z


# experts, groups, kept groups, k: of one or two lanes' places the last are behind the last expert, and the kept groups
# have one expert more than k or none (the first six); the same with more and fewer such places, and without groups
PLACES = [(63, 7, 1, 9), (63, 9, 1, 7), (63, 9, 2, 13), (63, 9, 2, 14), (126, 9, 1, 14), (126, 14, 1, 9), (62, 2, 1, 16), (60, 4, 1, 14),
          (8, 2, 1, 4), (12, 4, 2, 6), (255, 15, 1, 16), (510, 6, 1, 8), (1020, 15, 1, 14), (1023, 11, 1, 16), (7, 1, 1, 7), (15, 1, 1, 14),
          (63, 1, 1, 16), (3, 3, 1, 1), (16, 16, 9, 9), (513, 3, 2, 10)]


@pytest.mark.parametrize("E,G,top,k", PLACES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_places_behind_the_last_expert_are_not_chosen(E, G, top, k, scoring):
    T = 203
    for every in (1, 4, 7):
        z = near_pairs(T, E, E + k + every, every)
        g = torch.Generator().manual_seed(k)
        far = z.clone()  # the k-th choice at -inf, or far below the largest logit
        for t in range(0, T, every):
            far[t, torch.randperm(E, generator=g)[:E // 2 + 1]] = (-torch.inf, -70.0)[t % 2]
        last = z.clone()  # the last expert is the best of all
        last[:, -1] += 9.0
        for v in (z, far, last):
            kw = dict(scoring=scoring, groups=G, top_groups=top)
            check_route(v, k, renormalise=scoring == "softmax", **kw)
            bias = (torch.rand(E, generator=g) - 0.5) * 0.2
            for b in (bias, torch.zeros(E)):
                check_route(v, k, renormalise=False, bias=b, **kw)
                check_route(v.to(BF), k, renormalise=False, bias=b, **kw)
                if G > 1 and E // G > 1:
                    check_route(v, k, renormalise=False, bias=b, group_score="top2", **kw)
            if G > 1 and E // G > 1:
                check_route(v, k, renormalise=False, group_score="top2", **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,G,top,k", [(8, 4, 2, 3), (63, 7, 3, 5), (128, 8, 4, 8), (256, 16, 5, 12), (700, 10, 4, 6)])
def test_sums_of_both_infinities(E, G, top, k, scoring):
    """+inf beside nothing but -inf in a group: their sum is not a number and ranks as -inf."""
    each = E // G
    one = ((torch.rand(E, generator=torch.Generator().manual_seed(E)) - 0.5) * 0.2).view(G, each)
    one[G // 2] = -torch.inf
    one[G // 2, 1] = torch.inf
    for T, every in ((1, 1), (203, 203), (203, 4), (203, 1)):
        z = near_pairs(T, E, T + every, every)
        for bias in (one.flatten(), torch.where(torch.arange(E) % each == 1, torch.inf, -torch.inf),
                     torch.where(torch.arange(E) % 3 == 1, torch.inf, -torch.inf)):
            check_route(z, k, scoring=scoring, bias=bias, renormalise=False, groups=G, top_groups=top, group_score="top2")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("E,G,top,k", [(8, 4, 2, 3), (63, 7, 3, 5), (128, 8, 4, 8), (256, 16, 5, 12), (500, 4, 2, 16), (700, 10, 4, 6)])
def test_infinite_biases(E, G, top, k, scoring, dtype):
    """Groups with no, one or two experts that a bias of -inf leaves, and experts that a bias of +inf or NaN stands at."""
    each = E // G
    g = torch.Generator().manual_seed(E)
    finite = (torch.rand(E, generator=g) - 0.5) * 0.2
    biases = []
    for left in (0, 1, 2):
        b = finite.clone().view(G, each)
        b[1, left:] = -torch.inf
        b[G - 1, :max(0, each - left)] = -torch.inf
        biases.append(b.flatten())
        b = b.clone()
        b[0, 1:] = torch.nan
        biases.append(b.flatten())
    for n in (1, 2):
        b = finite.clone()
        b[E - n:] = torch.inf
        biases.append(b)
    biases += [torch.full((E,), -torch.inf), torch.full((E,), torch.inf),
               torch.where(torch.arange(E) % each == 0, finite, -torch.inf), torch.where(torch.arange(E) % each < 2, finite, -torch.inf),
               torch.where(torch.arange(E) % 5 == 1, 3e38, -3e38), torch.where(torch.arange(E) % 5 == 1, torch.inf, finite * 1e38)]
    for T, every in ((1, 1), (203, 203), (203, 4), (203, 1)):
        z = near_pairs(T, E, T + every, every).to(dtype)
        for b in biases:
            for group_score in ("top2", "max"):
                check_route(z, k, scoring=scoring, bias=b, renormalise=False, groups=G, top_groups=top, group_score=group_score)
            check_route(z, k, scoring=scoring, bias=b, renormalise=False)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("E,G,top,k", [(8, 4, 2, 3), (63, 7, 3, 5), (128, 8, 4, 8), (700, 10, 4, 6)])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_with_nan_logits(E, G, top, k, biased, dtype):
    """NaN logits that leave a group no, one or two experts; a NaN ranks as -inf."""
    T, each = 203, E // G
    for every in (T, 4, 1):
        z = near_pairs(T, E, every, every).to(dtype)
        for t in range(T):
            group = z[t, (t % G) * each:(t % G + 1) * each]
            group[t // G % 3:] = torch.nan
            if t % 5 == 0:
                z[t, 0] = torch.inf if t % 2 else -torch.inf
        bias = (torch.rand(E, generator=torch.Generator().manual_seed(E)) - 0.5) * 0.2 if biased else None
        for group_score in ("top2", "max"):
            kw = dict(scoring="sigmoid", groups=G, top_groups=top, group_score=group_score)
            r = route(z.to(DEV), k, selection_bias=None if bias is None else bias.to(DEV), **kw)
            assert torch.equal(r.ids.cpu().long(), R.choose(z, k, "sigmoid", bias, G, top, group_score))


@pytest.mark.parametrize("E", [40, 600])
def test_gradient_of_small_sigmoids(E):
    """Renormalised weights do not depend on how small their sum is, nor does what 1/sum is multiplied with."""
    T, k = 50, 6
    g = torch.Generator().manual_seed(E)
    for low in (-86.0, -70.0, -50.0):
        z = low + torch.rand(T, E, generator=g)
        ids = R.choose(z, k)
        for size in (1e-3, 1.0, 3e4):
            dw = torch.randn(T, k, generator=g) * size
            want, bound = R.gradient(dw, z, ids, "sigmoid")
            got = route_gradient(dw.to(DEV), z.to(DEV), ids.to(DEV, torch.int32), scoring="sigmoid")
            assert_within(got, want, bound, f"low {low}, size {size}")
