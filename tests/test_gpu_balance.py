"""netra_moe.balance (per-expert counts, balance loss and gradient) on the GPU
against the float64 formulas.

Bounds of the fp32 loss and gradient (u = 2^-24). With d = z - max(z) rounded
once (|d| u), p's exponent is off by at most (|d| + 4) u relative (d <= 104
matters; beyond, p < 2^-149), its sum over E adds (6 + E / 64) u, the division
1, f 3: a p is within (|d| + 20 + E / 64) u of itself, s within twice that of
its magnitude, and p (f - s) within four times that of p (f + s). Terms below
2^-126 may lose all of it: an absolute 2^-125 E f."""
import numpy as np
import pytest
import torch

import layers_case as C
from conftest import gpu_available
from netra_moe import balance as B

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32


def routing(T, E, K, seed, extra=0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E + extra, generator=g) * 2 + torch.randn(E + extra, generator=g)).to(dtype)
    ids = torch.topk(logits[:, :E].float(), K, dim=1).indices.to(torch.int32)
    if extra:
        ids = torch.cat([ids, torch.full((T, extra), E, dtype=torch.int32)], 1)
    return logits, ids.contiguous()


def check(r, logits, counts, coefficient=1.0, **kw):
    loss, grad, p, f, s, scale = C.balance(logits, counts, coefficient=coefficient, **kw)
    E = logits.shape[1]
    n = (104 + 20 + E / 64) * C.U
    tiny = 2.0 ** -125 * E * float(f.max()) * abs(scale)
    assert abs(float(r.loss) - loss) <= abs(loss) * 4 * n + tiny
    if r.grad is not None:
        assert r.grad.dtype == logits.dtype
        C.assert_within(r.grad, grad, 4 * n * p * (f + s) * abs(scale) + tiny, "gradient")


COUNTS = [(1, 1, 1), (1, 16, 2), (16, 16, 2), (64, 256, 8), (65, 257, 5), (700, 60, 6), (1025, 512, 3),
          (4096, 256, 8), (20001, 8, 2), (30000, 1024, 4), (9000, 1000, 8)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,E,K", COUNTS)
def test_counts(T, E, K, masked):
    _, ids = routing(T, E, K, seed=T + E, extra=1)
    ids[::7, 0] = -1
    ids[::11, K - 1] = 2 ** 31 - 1
    mask = torch.rand(T, generator=torch.Generator().manual_seed(1)) < 0.6 if masked else None
    d = ids.to(DEV)
    got = B.expert_counts(d, E, mask=None if mask is None else mask.to(DEV))
    want = C.counts(ids, E, mask)
    assert got.dtype == torch.int32
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    B.expert_counts(d, E, mask=None if mask is None else mask.to(DEV), out=got, accumulate=True)
    np.testing.assert_array_equal(got.cpu().numpy(), 2 * want)


def test_counts_of_one_expert_and_of_nothing():
    ids = torch.zeros(50000, 8, dtype=torch.int32, device=DEV)
    assert B.expert_counts(ids, 4).tolist() == [400000, 0, 0, 0]
    assert B.expert_counts(ids[:0], 4).tolist() == [0] * 4
    assert B.expert_counts(ids, 4, mask=torch.zeros(50000, dtype=torch.bool, device=DEV)).tolist() == [0] * 4
    keep = torch.tensor([5, 6, 7, 8], dtype=torch.int32, device=DEV)
    assert B.expert_counts(ids[:0], 4, out=keep, accumulate=True).tolist() == [5, 6, 7, 8]


def test_counts_of_strided_ids():
    base = torch.full((300, 12), 3, dtype=torch.int32, device=DEV)
    base[:, 5:8] = torch.randint(0, 3, (300, 3), dtype=torch.int32, device=DEV)
    got = B.expert_counts(base[:, 5:8], 4).cpu().numpy()
    np.testing.assert_array_equal(got, C.counts(base[:, 5:8], 4))


BALANCE = [(1, 1, 1, 0), (1, 16, 2, 0), (2, 64, 4, 1), (16, 16, 2, 0), (17, 65, 3, 0), (64, 256, 8, 1), (300, 128, 4, 1),
           (1000, 129, 2, 0), (513, 500, 6, 1), (4096, 256, 8, 1), (777, 1024, 8, 0), (2049, 700, 5, 0), (9001, 33, 3, 1),
           (5, 3, 1, 0), (100, 62, 3, 0), (200, 99, 4, 1), (256, 128, 8, 0), (128, 250, 8, 1), (257, 16, 2, 0),
           (32, 1024, 8, 1), (33, 1023, 4, 0)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,E,K,extra", BALANCE)
def test_balance(T, E, K, extra, masked, dt):
    logits, ids = routing(T, E, K, seed=T * 3 + E, extra=extra, dtype=dt)
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
    if mask is not None:
        assert torch.all(r.grad.cpu()[~mask] == 0)
    given = B.balance_loss(z, counts=r.counts, mask=m, coefficient=0.3)
    assert torch.equal(given.loss, r.loss) and torch.equal(given.grad, r.grad)
    alone = B.balance_loss(z, ids.to(DEV), mask=m, coefficient=0.3, grad=False)
    assert alone.grad is None and torch.equal(alone.loss, r.loss)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_bias_and_counts_of_a_larger_job(dt):
    logits, _ = routing(200, 96, 4, seed=5, dtype=dt)
    bias = torch.randn(96, generator=torch.Generator().manual_seed(6)) * 3
    counts = torch.randint(0, 1 << 20, (96,), generator=torch.Generator().manual_seed(7), dtype=torch.int32)
    r = B.balance_loss(logits.to(DEV), counts=counts.to(DEV), bias=bias.to(DEV), coefficient=2.0)
    check(r, logits, counts.numpy(), 2.0, bias=bias)


def test_rows_that_the_mask_or_the_logits_leave_empty():
    logits, ids = routing(40, 32, 2, seed=8, dtype=F32)
    logits[5] = -torch.inf              # nothing left in the row
    logits[6, 3:] = -torch.inf          # three experts left
    logits[7] = torch.finfo(F32).min    # the lowest value everywhere: an even row
    logits[8, 1:] = torch.finfo(F32).min
    logits[9] = 3e38
    r = B.balance_loss(logits.to(DEV), ids.to(DEV))
    check(r, logits, C.counts(ids, 32))
    assert torch.all(r.grad[5] == 0)
    none = B.balance_loss(logits.to(DEV), ids.to(DEV), mask=torch.zeros(40, dtype=torch.bool, device=DEV))
    assert float(none.loss) == 0 and torch.all(none.grad == 0) and torch.all(none.counts == 0)
    gone = B.balance_loss(logits.to(DEV), torch.full_like(ids, -1).to(DEV))
    assert float(gone.loss) == 0 and torch.all(gone.grad == 0)
    empty = B.balance_loss(logits[:0].to(DEV), ids[:0].to(DEV))
    assert float(empty.loss) == 0 and empty.grad.shape == (0, 32) and torch.all(empty.counts == 0)


def test_nan_reaches_its_row_and_the_loss():
    logits, ids = routing(40, 80, 2, seed=9, dtype=F32)
    logits[4, 77], logits[5, 0], logits[6] = torch.nan, torch.inf, torch.nan
    r = B.balance_loss(logits.to(DEV), ids.to(DEV))
    bad = torch.isnan(r.grad).all(1).cpu()
    assert bad.nonzero().view(-1).tolist() == [4, 5, 6] and torch.isnan(r.loss)
    assert not torch.isnan(r.grad.cpu()[~bad]).any()


def test_gradient_against_differences():
    """Central differences of the float64 loss with the counts held fixed; step h
    leaves a third derivative's h^2 term and the loss's own rounding."""
    logits, ids = routing(6, 10, 2, seed=10, dtype=F32)
    r = B.balance_loss(logits.to(DEV), ids.to(DEV), coefficient=1.5)
    counts, h = C.counts(ids, 10), 1e-4
    grad = r.grad.cpu().double()
    for t in range(6):
        for e in range(10):
            z = logits.double()
            lo, hi = z.clone(), z.clone()
            lo[t, e] -= h
            hi[t, e] += h
            diff = (C.balance(hi, counts, coefficient=1.5)[0] - C.balance(lo, counts, coefficient=1.5)[0]) / (2 * h)
            # |third derivative of p f| <= 6 f_max p, f_max <= 10, scale 1.5 / 6
            assert abs(float(grad[t, e]) - diff) <= 10 * h * h * 2.5 + 1e-11 + 1e-5 * abs(diff) + 1e-7


def test_an_even_router_costs_the_coefficient():
    T, E = 64, 32
    ids = torch.arange(T * 2, dtype=torch.int32, device=DEV).view(T, 2) % E
    r = B.balance_loss(torch.zeros(T, E, device=DEV), ids, coefficient=0.25)
    assert float(r.loss) == 0.25 and torch.all(r.grad == 0)


def test_captured_graph_replays_beside_eager_work():
    logits, ids = routing(3000, 256, 8, seed=11, extra=1)
    z, d = logits.to(DEV), ids.to(DEV)
    B.balance_loss(z[:, :256], d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = B.balance_loss(z[:, :256], d, coefficient=0.1)
        c = B.expert_counts(d, 256)
    for i in range(4):
        logits, ids = routing(3000, 256, 8, seed=20 + i, extra=1)
        z.copy_(logits)
        d.copy_(ids)
        graph.replay()
        torch.cuda.synchronize()
        e = B.balance_loss(z[:, :256], d, coefficient=0.1)
        assert torch.equal(r.loss, e.loss) and torch.equal(r.grad, e.grad) and torch.equal(r.counts, e.counts)
        assert torch.equal(c, e.counts)


def test_two_streams_at_once():
    sets = [routing(T, 200, 4, seed=T) for T in (5000, 40, 900)]
    sets = [(a.to(DEV), b.to(DEV)) for a, b in sets]
    want = [B.balance_loss(a, b) for a, b in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in sets]
    for _ in range(5):
        got = []
        for st, (a, b) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(B.balance_loss(a, b))
        torch.cuda.synchronize()
        for r, w in zip(got, want):
            assert torch.equal(r.loss, w.loss) and torch.equal(r.grad, w.grad) and torch.equal(r.counts, w.counts)


def test_refusals():
    z = torch.zeros(4, 8, device=DEV)
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    for args, kw in [((z.half(), ids), {}), ((z.t(), ids), {}), ((z, ids.long()), {}), ((z, ids[:3]), {}), ((z,), {}),
                     ((z, ids), {"counts": torch.zeros(8, dtype=torch.int32, device=DEV)}),
                     ((z, ids), {"mask": torch.ones(3, dtype=torch.bool, device=DEV)}),
                     ((z, ids), {"bias": torch.zeros(7, device=DEV)}),
                     ((z,), {"counts": torch.zeros(8, device=DEV)}), ((z.cpu(), ids), {}),
                     ((torch.zeros(4, 1025, device=DEV), ids), {})]:
        with pytest.raises(ValueError):
            B.balance_loss(*args, **kw)
    for args, kw in [((ids, 0), {}), ((ids, 1025), {}), ((ids.cpu(), 8), {}), ((ids, 8), {"accumulate": True}),
                     ((ids[:, :0], 8), {}), ((ids, 8), {"out": torch.zeros(9, dtype=torch.int32, device=DEV)})]:
        with pytest.raises(ValueError):
            B.expert_counts(*args, **kw)
