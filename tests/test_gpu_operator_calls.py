"""Calls of the norm, the routing and the adapters that their documentation allows: from
several threads, in graphs that replay next to each other, behind a HIP error that
another call left, inputs larger than the caches, and rows that are views."""
import threading

import pytest
import torch

import adapters_case as A
import norm_case as N
from conftest import gpu_available
from layers_case import assert_within
from layers_case import weights as fp8_weights
from netra_moe.adapters import LowRankAdapters, make_plan
from netra_moe.linear import BlockLinear
from netra_moe.norm import rms_norm, rms_norm_gradients
from netra_moe.routing import route, route_gradient
from test_layers_errors import INVALID_DEVICE, hip

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = torch.device("cuda", 0)


class Step:
    """A norm, a projection with adapters, the routing, and the gradients of both."""
    L = 6

    def __init__(self, T, H=640, n=512, E=96, seed=1):
        g = torch.Generator().manual_seed(seed)
        q, s, _ = fp8_weights(n, H, seed)
        a, b, scale = A.adapters(self.L, 24, H, n, seed)
        self.proj = BlockLinear(q.to(DEV), s.to(DEV))
        self.adapters = LowRankAdapters(a.to(DEV), b.to(DEV), scale.to(DEV))
        self.x, self.stream, self.dy = (torch.randn(T, H, generator=g).to(BF).to(DEV) for _ in range(3))
        self.w = torch.rand(H, generator=g).to(DEV)
        self.z = torch.randn(T, E, generator=g).to(DEV)
        self.bias = (torch.rand(E, generator=g) * 0.1).to(DEV)
        self.dweights = torch.randn(T, 4, generator=g).to(DEV)
        self.ids = torch.randint(-1, self.L, (T,), generator=g, dtype=torch.int32).to(DEV)

    def run(self):
        n = rms_norm(self.x, self.w, residual=self.stream, codes="tiles")
        plan = make_plan(self.ids, self.L)
        y = self.adapters.add(self.proj.forward_codes(n.codes, n.scale, len(self.x)), n.y, plan)
        kw = dict(scoring="sigmoid", scale=2.0)
        r = route(self.z, 4, selection_bias=self.bias, groups=8, top_groups=4, group_score="top2", **kw)
        return [n.residual, n.y, y, r.ids, r.weights, route_gradient(self.dweights, self.z, r.ids, **kw),
                *rms_norm_gradients(self.dy, n.residual, self.w, residual_gradient=self.stream)]


def same(a, b):
    return all(torch.equal(v, w) for v, w in zip(a, b, strict=True))


def test_calls_from_several_threads():
    steps = [Step(T, seed=i) for i, T in enumerate((1, 17, 130, 1200))]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    got = [[] for _ in steps]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            for _ in range(10):
                got[i].append(steps[i].run())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert len(runs) == 10 and all(same(r, w) for r in runs)


def test_two_graphs_replay_at_once():
    graphs = []
    for i, T in enumerate((300, 900)):
        step = Step(T, seed=20 + i)
        eager = step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step.run()
        graphs.append((graph, torch.cuda.Stream(DEV), out, eager, step))
    for _ in range(5):
        for _, _, out, _, _ in graphs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream, _, _, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, eager, _ in graphs:
            assert same(out, eager)


def test_calls_run_behind_a_stale_error_and_leave_it_to_the_caller():
    step = Step(70, seed=5)
    want = step.run()
    torch.cuda.synchronize()
    assert hip("hipSetDevice", 12345) == INVALID_DEVICE
    try:
        got = step.run()
        assert hip("hipPeekAtLastError") == INVALID_DEVICE
    finally:
        hip("hipGetLastError")
    assert same(got, want)


# one length of each kernel's
@pytest.mark.parametrize("H", [512, 1000, 2048, 4096, 8191, 16384])
@pytest.mark.parametrize("types", [(BF, BF), (BF, F), (F, BF), (F, F)])
def test_norm_of_more_than_the_caches_hold(H, types):
    """A row does not depend on the others: the same bits as of a call of a few rows. dw by the formula."""
    gen = torch.Generator(device=DEV).manual_seed(H)
    size = {BF: 2, F: 4}
    row = H * (size[types[0]] + 2 * size[types[1]])  # what the gradients move at least; the norm moves more
    T = (1 << 28) // row + 37
    x, stream = (torch.randn(T, H, generator=gen, device=DEV).to(t) for t in types)
    w = torch.rand(H, generator=gen, device=DEV)
    n = rms_norm(x, w, residual=stream, codes="rows")
    dr, dw = rms_norm_gradients(x, n.residual, w)
    for rows in (slice(0, 40), slice(T - 40, T)):
        few = rms_norm(x[rows], w, residual=stream[rows], codes="rows")
        assert torch.equal(n.y[rows], few.y) and torch.equal(n.residual[rows], few.residual)
        assert torch.equal(n.codes[rows].view(torch.uint8), few.codes.view(torch.uint8)) and torch.equal(n.scale[rows], few.scale)
        assert torch.equal(dr[rows], rms_norm_gradients(x[rows], few.residual, w)[0])
    want, bound = torch.zeros(H, dtype=torch.float64, device=DEV), torch.zeros(H, dtype=torch.float64, device=DEV)
    for at in range(0, T, 4096):
        r = n.residual[at:at + 4096].double()
        t = x[at:at + 4096].double() * r / (r.square().mean(1, keepdim=True) + 1e-6).sqrt()
        want += t.sum(0)
        bound += t.abs().sum(0)
    assert_within(dw, want.cpu(), ((T + 60) * N.U * bound).cpu(), "dw")


def test_views_of_one_row_and_one_column():
    """Strides that a dimension of one leaves open are not followed."""
    base = torch.randn(300, 7, device=DEV)
    w = torch.rand(300, device=DEV)
    one = torch.as_strided(base, (1, 300), (1, 1))
    n = rms_norm(one, w, out_type=F)
    assert torch.equal(n.y, rms_norm(base.flatten()[:300].clone()[None], w, out_type=F).y)
    dx, dw = rms_norm_gradients(one, one, w)
    assert torch.equal(dx, rms_norm_gradients(one.clone(), one.clone(), w)[0]) and torch.isfinite(dw).all()
    z = torch.as_strided(base, (1, 16), (0, 1))
    assert torch.equal(route(z, 4).ids, route(z.clone(), 4).ids)
    column = base[:, 3:4]
    n = rms_norm(column, w[:1], out_type=F)
    assert torch.equal(n.y, rms_norm(column.contiguous(), w[:1], out_type=F).y)
    assert torch.equal(route(column, 1).weights, torch.ones(300, 1, device=DEV))


# T, adapters, rank, K, N: y and out of more than 256 MiB, of each tile and rank
ONCE = [(7000, 3, 16, 128, 10001), (7000, 9, 20, 128, 9999), (7001, 3, 64, 200, 10240), (7000, 60, 100, 200, 10000),
        (9000, 3, 16, 128, 10001), (9001, 9, 20, 128, 9999), (8192, 3, 64, 200, 10240), (9000, 60, 100, 200, 10000)]


@pytest.mark.parametrize("T,L,r,K,N", ONCE)
def test_adapters_of_more_than_the_caches_hold(T, L, r, K, N):
    """A row does not depend on the others; the first and last rows by the formula."""
    a, b, s = A.adapters(L, r, K, N, r)
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    gen = torch.Generator(device=DEV).manual_seed(T)
    x, y = (torch.randn(T, n, generator=gen, device=DEV).to(BF) for n in (K, N))
    ids = torch.randint(-1, L, (T,), generator=gen, device=DEV, dtype=torch.int32)
    got = lora.add(y, x, lora.plan(ids))
    for rows in (slice(0, 50), slice(T - 50, T)):
        want, bound = A.add(y[rows].cpu(), x[rows].cpu(), a, b, s, ids[rows].cpu())
        assert_within(got[rows], want, bound)
    order = torch.randperm(T, generator=gen, device=DEV)
    again = lora.add(y[order], x[order], lora.plan(ids[order]))
    assert torch.equal(again, got[order])
    assert torch.equal(got[ids < 0], y[ids < 0])
    assert lora.add(y, x, lora.plan(ids), y) is y and torch.equal(y, got)


def test_a_projection_refuses_another_batchs_plan_before_it_writes():
    step = Step(40)
    out = torch.zeros(40, 512, dtype=BF, device=DEV)
    for plan in (make_plan(step.ids[:39].contiguous(), Step.L), make_plan(step.ids, Step.L + 1), None):
        with pytest.raises(ValueError):
            step.proj.forward(step.x, out, adapters=step.adapters, plan=plan)
    torch.cuda.synchronize()
    assert not out.any()
    assert step.proj.forward(step.x, out, adapters=step.adapters, plan=make_plan(step.ids, Step.L)) is out and out.any()
