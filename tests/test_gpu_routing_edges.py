"""netra_moe.routing where the kept groups hold hardly more experts than are chosen (forms and bounds of routing_case.py)."""
import pytest
import torch

from conftest import gpu_available
from test_gpu_routing import check_route

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32


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
