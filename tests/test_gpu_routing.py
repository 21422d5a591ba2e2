"""netra_moe.routing on the GPU against its 64-bit forms (routing_case.py)."""
import pytest
import torch

import routing_case as R
from conftest import gpu_available
from layers_case import assert_within
from netra_moe.balance import balance_loss, expert_counts
from netra_moe.routing import route, route_gradient

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = "cuda:0"
GROUPED = dict(groups=4, top_groups=2)
# tokens, experts, k, groups
SIZES = [(1, 1, 1, 1), (3, 2, 2, 2), (5, 8, 2, 4), (64, 64, 8, 8), (7, 65, 3, 5), (33, 100, 10, 10), (130, 128, 8, 4), (65, 256, 8, 8),
         (6, 257, 16, 1), (9, 300, 6, 3), (1000, 500, 6, 4), (2, 512, 15, 16), (5, 513, 9, 9), (11, 1000, 8, 8), (3, 1024, 16, 16),
         (70001, 16, 2, 4)]


def check_route(z, k, mask=None, bias=None, scoring="softmax", renormalise=True, scale=1.0, shared=False, groups=1, top_groups=None,
                group_score="max"):
    r = route(z.to(DEV), k, scoring=scoring, selection_bias=None if bias is None else bias.to(DEV), groups=groups,
              top_groups=top_groups, group_score=group_score, renormalise=renormalise, scale=scale, shared=shared,
              mask=None if mask is None else mask.to(DEV))
    E = z.shape[1] - shared
    live = torch.ones(len(z), dtype=torch.bool) if mask is None else mask
    ids = R.choose(z[live][:, :E], k, scoring, bias, groups, groups if top_groups is None else top_groups, group_score)
    assert torch.equal(r.ids[:, :k].cpu()[live].long(), ids)
    if shared:
        assert (r.ids[:, k].cpu()[live] == E).all()
    assert (r.ids.cpu()[~live] == -1).all() and not r.weights.cpu()[~live].any()
    want, bound = R.weights(z[live], ids, scoring, renormalise, scale, shared)
    assert_within(r.weights.cpu()[live], want, bound, "weights")
    return r


@pytest.mark.parametrize("T,E,k,G", SIZES)
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("scoring,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route(T, E, k, G, dtype, scoring, renormalise):
    shared = (T + E) % 2 == 1 and k < 16
    z = R.inputs(T, E, T + E, dtype, shared)
    mask = torch.arange(T) % 3 != 1 if E % 2 else None
    top = max(1, -(-k * G // E), G // 2)
    kw = dict(scoring=scoring, renormalise=renormalise, scale=2.5, shared=shared, mask=mask)
    check_route(z, k, **kw)
    check_route(z, k, groups=G, top_groups=top, **kw)
    if E // G >= 2:
        bias = (torch.rand(E, generator=torch.Generator().manual_seed(E)) - 0.5) * 0.2
        check_route(z, k, groups=G, top_groups=top, group_score="top2", **kw)
        check_route(z, k, groups=G, top_groups=top, group_score="top2", bias=bias, **kw)
        check_route(z, k, groups=G, top_groups=top, bias=bias, **kw)
        check_route(z, k, bias=bias * 0.0, **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [32, 256, 400, 700])
def test_ties_go_to_the_lower_index(scoring, E):
    g = torch.Generator().manual_seed(E)
    z = torch.randint(-2, 3, (200, E), generator=g).to(BF)
    check_route(z, 8, scoring=scoring)
    check_route(z, 8, scoring=scoring, groups=4, top_groups=2)
    check_route(z, 8, scoring=scoring, groups=4, top_groups=2, group_score="top2")
    check_route(z, 8, scoring=scoring, bias=torch.zeros(E))
    check_route(z, 8, scoring=scoring, bias=torch.randint(0, 2, (E,), generator=g) * 0.25, groups=4, top_groups=3)
    check_route(torch.zeros(5, E), 8, scoring=scoring, bias=torch.zeros(E), groups=4, top_groups=2, group_score="top2")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("grouped", [False, True])
def test_scores_that_differ_by_less_than_fp32_tells(scoring, grouped):
    """Every expert's bias brings its score to within an fp32 rounding of the same value: which is larger
    shows only in 64 bits."""
    T, E = 300, 128
    z = R.inputs(1, E, 5, F).expand(T, E).clone()
    s = R.scores(z[:1].double(), scoring)[0]
    bias = (0.75 - s).float()
    # tokens with a few experts moved by their neighbours' last bits
    z = z * (1 + (torch.randint(-2, 3, (T, E), generator=torch.Generator().manual_seed(2)) * 2.0 ** -23))
    kw = dict(groups=8, top_groups=3, group_score="top2") if grouped else {}
    check_route(z, 8, scoring=scoring, bias=bias, **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,G", [(48, 4), (520, 8)])
def test_infinities_and_nan(scoring, E, G):
    z = R.inputs(40, E, 9, F)
    z[1] = -torch.inf
    z[2, 5:] = -torch.inf
    z[3, : E // 2] = -torch.inf
    z[4] = 1000.0
    z[5] = -1000.0
    z[6, 7] = 90.0
    z[8] = torch.linspace(-1e4, 1e4, E)
    for kw in (dict(), dict(renormalise=False), dict(groups=G, top_groups=2), dict(bias=torch.zeros(E)),
               dict(groups=G, top_groups=2, group_score="top2")):
        if scoring == "sigmoid" and kw.get("renormalise", True):
            # (sums of sigmoids that underflow in fp32 are 0 by definition)
            rows = [t for t in range(40) if t not in (2, 5, 8)]
            check_route(z[rows], 8, scoring=scoring, **kw)
        else:
            check_route(z, 8, scoring=scoring, **kw)
    # a NaN is chosen last, ids stay distinct and in range
    z[0, 3] = torch.nan
    z[7] = torch.nan
    for kw in (dict(), dict(groups=G, top_groups=3), dict(selection_bias=torch.zeros(E, device=DEV))):
        r = route(z.to(DEV), 8, scoring=scoring, **kw)
        ids = r.ids.cpu()
        assert ((ids >= 0) & (ids < E)).all() and all(len(set(row.tolist())) == 8 for row in ids)
        if scoring == "sigmoid" or "selection_bias" not in kw:  # (a NaN makes every softmax score of its row one)
            assert 3 not in ids[0].tolist()
        assert torch.isfinite(r.weights.cpu()[9:]).all()


@pytest.mark.parametrize("T,E,k,G", SIZES)
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("scoring,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient(T, E, k, G, dtype, scoring, renormalise):
    shared = (T + E) % 2 == 1 and k < 16
    z = R.inputs(T, E, T + E, dtype, shared)
    g = torch.Generator().manual_seed(T)
    ids = R.choose(z[:, :E], k)
    if shared:
        ids = torch.cat([ids, torch.full((T, 1), E)], 1)
    dw = torch.randn(T, k + shared, generator=g)
    mask = torch.rand(T, generator=g) < 0.7 if E % 2 else None
    kw = dict(scoring=scoring, renormalise=renormalise, scale=2.5, shared=shared)
    args = (dw.to(DEV), z.to(DEV), ids.to(DEV, torch.int32))
    got = route_gradient(*args, mask=None if mask is None else mask.to(DEV), **kw)
    want, bound = R.gradient(dw, z, ids, **kw)
    if mask is not None:
        want, bound = want * mask[:, None], bound * mask[:, None]
    assert_within(got, want, bound, "grad")
    old = torch.randn(T, E + shared, generator=g).to(dtype)
    out = old.to(DEV)
    route_gradient(*args, mask=None if mask is None else mask.to(DEV), out=out, accumulate=True, **kw)
    assert_within(out, want + old.double(), bound + 2 * R.U * (want.abs() + old.double().abs()), "accumulated")


@pytest.mark.parametrize("scoring,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("E", [40, 600])
def test_gradient_of_dropped_and_repeated_slots(scoring, renormalise, E):
    T, k = 60, 7
    z = R.inputs(T, E, 2, F, True, spread=4.0)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, E, (T, k + 1), generator=g)
    ids[:, 3], ids[::2, 5] = ids[:, 0], ids[::2, 0]  # the same expert in two and three slots
    ids[5], ids[6, 1], ids[7, 2] = -1, E, 1 << 30
    ids[8] = 1
    dw = torch.randn(T, k + 1, generator=g)
    kw = dict(scoring=scoring, renormalise=renormalise, shared=True)
    want, bound = R.gradient(dw, z, ids, **kw)
    got = [route_gradient(dw.to(DEV), z.to(DEV), ids.to(DEV, torch.int32), **kw) for _ in range(3)]
    assert_within(got[0], want, bound)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_gradient_where_one_expert_has_almost_everything():
    z = torch.full((4, 64), -3.0)
    z[:, 9] = torch.tensor([5.0, 12.0, 20.0, 60.0])
    ids = R.choose(z, 2)
    dw = torch.tensor([[1.0, 1.0 + 2.0 ** -10]]).expand(4, 2)
    for renormalise in (True, False):
        for scoring in ("softmax", "sigmoid"):
            want, _ = R.gradient(dw, z, ids, scoring, renormalise)
            got = route_gradient(dw.contiguous().to(DEV), z.to(DEV), ids.to(DEV, torch.int32), scoring=scoring, renormalise=renormalise)
            # relative to itself, not to |v_i| + |v_j|: 100 u and 4 |z - m| u = 252 u
            chosen = torch.gather(want, 1, ids)
            assert_within(torch.gather(got.cpu(), 1, ids), chosen, 360 * R.U * chosen.abs() + 1e-36)


@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_of_wider_matrices(dtype):
    """Logits and gradients as column slices at odd places; their neighbours stay as they were."""
    T, E = 37, 99
    wide = R.inputs(T, 120, 3, dtype).to(DEV)
    z = wide[:, 3:3 + E + 1]
    r = route(z, 5, shared=True, scoring="sigmoid")
    ids = R.choose(z[:, :E].cpu(), 5)
    assert torch.equal(r.ids[:, :5].cpu().long(), ids)
    out = torch.full((T, 131), 7.0, dtype=dtype, device=DEV)
    dw = torch.randn(T, 9, device=DEV)[:, 2:8]
    ids9 = torch.zeros((T, 8), dtype=torch.int32, device=DEV)
    ids9[:, 1:7] = r.ids
    route_gradient(dw, z, ids9[:, 1:7], shared=True, scoring="sigmoid", out=out[:, 5:5 + E + 1])
    want, bound = R.gradient(dw, z, r.ids, "sigmoid", shared=True)
    assert_within(out[:, 5:5 + E + 1], want, bound)
    assert (out[:, :5] == 7).all() and (out[:, 5 + E + 1:] == 7).all()


def test_a_step_with_counts_and_balance_loss_another_stream_and_a_graph():
    """The run of operators of a training step's router, eager on another stream, and captured and replayed."""
    T, E, k = 300, 96, 4
    z = R.inputs(T, E, 6, F).to(DEV)
    bias = (torch.rand(E, device=DEV) - 0.5) * 0.1
    dw = torch.randn(T, k, device=DEV)
    mask = torch.rand(T, device=DEV) < 0.8

    def step():
        r = route(z, k, scoring="sigmoid", selection_bias=bias, groups=8, top_groups=3, group_score="top2", mask=mask)
        b = balance_loss(z, r.ids, mask=mask, coefficient=0.01)
        aux = b.grad.clone()
        route_gradient(dw, z, r.ids, scoring="sigmoid", mask=mask, out=b.grad, accumulate=True)
        return r.ids, r.weights, expert_counts(r.ids, E), b.counts, b.grad, aux

    want = step()
    assert torch.equal(want[2], want[3]) and int(want[2].sum()) == k * int(mask.sum())
    ids = R.choose(z.cpu(), k, "sigmoid", bias, 8, 3, "top2")
    assert torch.equal(want[0].cpu()[mask.cpu()].long(), ids[mask.cpu()])
    g, bound = R.gradient(dw, z, want[0], "sigmoid")
    g, bound = g * mask.cpu()[:, None], bound * mask.cpu()[:, None]
    total = g + want[5].cpu().double()
    assert_within(want[4], total, bound + 2 * R.U * (g.abs() + want[5].cpu().double().abs()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        if n:
            z.copy_(torch.randn_like(z))
            want = step()
        for h in held:
            h.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=17), dict(k=9), dict(k=2, groups=3), dict(k=5, groups=4, top_groups=2), dict(k=2, scoring="relu"),
                                dict(k=2, groups=2, group_score="sum"), dict(k=2, groups=8, top_groups=4, group_score="top2"),
                                dict(k=2, mask=torch.ones(3, dtype=torch.bool)), dict(k=2, selection_bias=torch.zeros(8)),
                                dict(k=2, top_groups=2)])
def test_refusals(kw):
    with pytest.raises((ValueError, RuntimeError)):
        route(torch.zeros(4, 8, device=DEV), kw.pop("k"), **kw)


def test_gradient_refusals():
    z, ids, dw = torch.zeros(4, 8, device=DEV), torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.zeros(4, 2, device=DEV)
    for args, kw in [((dw.half(), z, ids), {}), ((dw, z, ids.long()), {}), ((dw, z, ids[:3]), {}), ((dw, z, ids), dict(out=z)),
                     ((dw, z, ids), dict(accumulate=True)), ((dw, z.half(), ids), {}), ((dw[:, :0], z, ids[:, :0]), {}),
                     ((dw, z, ids), dict(out=torch.zeros(4, 8, device=DEV, dtype=BF)))]:
        with pytest.raises((ValueError, RuntimeError)):
            route_gradient(*args, **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [20, 128, 300, 700])
@pytest.mark.parametrize("k", [8, 13, 14, 15, 16])
def test_near_scores_on_both_sides_of_the_last_choice(scoring, E, k):
    """The k-th and the next few experts are equal, or apart by less than fp32 tells or by a little more; in some tokens
    one lane has most of them."""
    T = 240
    g = torch.Generator().manual_seed(E + k)
    z = torch.randn(T, E, generator=g) * 0.1
    for t in range(T):
        order = torch.arange(E) if t % 3 == 0 else torch.randperm(E, generator=g)
        z[t, order[:k - 2]] += 3.0
        step = (0.0, 2.0 ** -23, 2.0 ** -21, 2.0 ** -19)[t % 4]
        near = order[k - 2:k + 2]
        z[t, near] = 2.0 + step * torch.randint(0, 3, (len(near),), generator=g)
    check_route(z, k, scoring=scoring)
    check_route(z, k, scoring=scoring, bias=torch.zeros(E))
    check_route(z, k, scoring=scoring, bias=(torch.rand(E, generator=g) * 2.0 ** -18))
    check_route(z.to(BF), k, scoring=scoring, bias=torch.zeros(E))
    if E % 4 == 0:
        check_route(z, k, scoring=scoring, groups=4, top_groups=4 if E == 20 else 3, group_score="top2")
