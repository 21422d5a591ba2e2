"""netra_moe.adapters on the GPU against its 64-bit form (adapters_case.py)."""
import pytest
import torch

import adapters_case as C
from conftest import gpu_available
from layers_case import assert_within
from layers_case import weights as fp8_weights
from netra_moe.adapters import LowRankAdapters, make_plan
from netra_moe.linear import BlockLinear

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = "cuda:0"


def batch(T, K, N, seed, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g)
    x[:, 3::37] *= 20.0
    return x.to(dtype), torch.randn(T, N, generator=g).to(BF)


def ids_of(T, L, chunk, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-1, L, (-(-T // chunk),), generator=g).repeat_interleave(chunk)[:T].to(torch.int32)


# T, L, r, K, N, tokens that follow each other with one adapter
SIZES = [(1, 1, 1, 1, 1, 1), (1, 4, 8, 2048, 2048, 1), (2, 2, 16, 64, 64, 1), (3, 1, 17, 100, 70, 3), (16, 5, 4, 128, 63, 1),
         (17, 1, 16, 129, 65, 17), (64, 32, 16, 512, 500, 1), (50, 7, 33, 1111, 130, 9), (203, 3, 12, 257, 300, 41),
         (100, 1000, 6, 96, 80, 1), (300, 2, 128, 333, 777, 150), (1025, 4, 64, 200, 129, 100), (2000, 9, 100, 130, 257, 33),
         (1500, 1, 32, 64, 2050, 1500), (40, 3, 20, 8192, 40, 5), (7, 2, 50, 130, 600, 1), (33, 3, 100, 300, 1030, 4), (5, 2, 128, 512, 512, 1),
         (600, 3, 40, 640, 520, 7), (1100, 2, 90, 1030, 1500, 13), (5000, 1024, 5, 40, 33, 2), (8200, 3, 100, 330, 300, 700), (8192, 9, 24, 130, 600, 11), (9000, 2, 64, 256, 129, 1), (8500, 120, 16, 70, 512, 5)]


@pytest.mark.parametrize("T,L,r,K,N,chunk", SIZES)
@pytest.mark.parametrize("dtype", [BF, F])
def test_add(T, L, r, K, N, chunk, dtype):
    a, b, s = C.adapters(L, r, K, N, T + r, F if T % 2 else BF)
    x, y = batch(T, K, N, T, dtype)
    ids = ids_of(T, L, chunk, T + 1)
    if T == 1:
        ids[:] = L - 1
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    plan = lora.plan(ids.to(DEV))
    yd, xd = y.to(DEV), x.to(DEV)
    got = lora.add(yd, xd, plan)
    want, bound = C.add(y, x, a, b, s, ids)
    assert_within(got, want, bound)
    assert torch.equal(yd.cpu(), y)
    none = (ids < 0) | (ids >= L)
    assert torch.equal(got.cpu()[none], y[none])
    assert lora.add(yd, xd, plan, yd) is yd  # in place: the same bits
    assert torch.equal(yd, got)


@pytest.mark.parametrize("T,L", [(1, 1), (63, 3), (64, 64), (1000, 1), (1024, 1024), (1025, 32), (5000, 7), (9000, 5), (70000, 500)])
def test_plan(T, L):
    """Every token once, by adapter and within one in the batch's order, in tiles of one adapter."""
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-2, L + 2, (T,), generator=g).to(torch.int32)
    ids[T // 2:] = ids[T // 2]
    words = make_plan(ids.to(DEV), L).data.cpu().view(torch.int32)
    of = torch.where((ids < 0) | (ids >= L), L, ids)
    assert words[:4].tolist()[1:] == [T, L, 0]
    assert torch.equal(words[4:4 + T].long(), torch.sort(of, stable=True).indices)
    tile = 32 if T >= 8192 and T // 64 >= L else 16
    start = 4 + -(-T // 4) * 4
    want, at = [], 0
    for l, n in enumerate(torch.bincount(of, minlength=L + 1).tolist()):
        want += [[l, at + i, min(tile, n - i), 0] for i in range(0, n, tile)]
        at += n
    assert words[0] == len(want)
    assert words[start:start + 4 * len(want)].view(-1, 4).tolist() == want


@pytest.mark.parametrize("ids", [[-1] * 40, [2] * 40, [7, -5, 3] * 13 + [1 << 30]])
def test_batches_of_one_adapter_or_none(ids):
    ids = torch.tensor(ids, dtype=torch.int32)
    a, b, s = C.adapters(3, 9, 150, 90, 4)
    x, y = batch(len(ids), 150, 90, 5)
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    got = lora.add(y.to(DEV), x.to(DEV), lora.plan(ids.to(DEV)))
    want, bound = C.add(y, x, a, b, s, ids)
    assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides_alignment_and_neighbours(dtype):
    T, L, r, K, N = 45, 4, 10, 301, 133
    a, b, s = C.adapters(L, r, K, N, 7)
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    ids = ids_of(T, L, 2, 3)
    plan = lora.plan(ids.to(DEV))
    g = torch.Generator().manual_seed(8)
    xw = torch.randn(T, 311, generator=g).to(dtype).to(DEV)
    yw = torch.randn(T, 140, generator=g).to(BF).to(DEV)
    x, y = xw[:, 5:5 + K], yw[:, 3:3 + N]
    want, bound = C.add(y, x, a, b, s, ids)
    out = torch.full((T, 151), 7.0, dtype=BF, device=DEV)
    lora.add(y, x, plan, out[:, 9:9 + N])
    assert_within(out[:, 9:9 + N], want, bound)
    assert (out[:, :9] == 7).all() and (out[:, 9 + N:] == 7).all()
    kept = yw.clone()
    lora.add(y, x, plan, y)
    assert_within(y, want, bound)
    assert torch.equal(yw[:, :3], kept[:, :3]) and torch.equal(yw[:, 3 + N:], kept[:, 3 + N:])


def test_infinities_and_nan_keep_to_their_rows():
    T, L, r, K, N = 40, 3, 5, 200, 96
    a, b, s = C.adapters(L, r, K, N, 1)
    b = b.abs() + 0.125
    a = a.abs() + 0.0625
    x, y = batch(T, K, N, 2)
    x[3, 7], x[4, 9], y[5, 2] = torch.inf, torch.nan, torch.inf
    ids = torch.arange(T, dtype=torch.int32) % 4 % 3
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    got = lora.add(y.to(DEV), x.to(DEV), lora.plan(ids.to(DEV))).cpu()
    want, bound = C.add(y, x, a, b, s, ids)
    assert (got[3] == torch.inf).all() and torch.isnan(got[4]).all() and got[5, 2] == torch.inf
    rows = [t for t in range(T) if t not in (3, 4, 5)]
    assert_within(got[rows], want[rows], bound[rows])


def test_ranks_of_their_own():
    pairs = []
    for i, r in enumerate((4, 16, 9)):
        a, b, _ = C.adapters(1, r, 140, 77, i)
        pairs.append((a[0].to(DEV), b[0].to(DEV)))
    lora = LowRankAdapters.from_pairs(pairs)
    assert (lora.count, lora.rank) == (3, 16)
    x, y = batch(30, 140, 77, 3)
    ids = ids_of(30, 3, 1, 4)
    got = lora.add(y.to(DEV), x.to(DEV), lora.plan(ids.to(DEV))).cpu()
    for l, (a, b) in enumerate(pairs):
        t = ids == l
        want, bound = C.add(y[t], x[t], a[None], b[None], torch.ones(1), torch.zeros(int(t.sum())))
        assert_within(got[t], want, bound)


def test_a_row_does_not_depend_on_its_neighbours():
    """The same token alone and in a batch of others: the same bits (k's splits apart, which go by the batch's size)."""
    a, b, s = C.adapters(4, 16, 600, 200, 5)
    x, y = batch(33, 600, 200, 6)
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    ids = ids_of(33, 4, 1, 7)
    whole = lora.add(y.to(DEV), x.to(DEV), lora.plan(ids.to(DEV)))
    turned = torch.randperm(33, generator=torch.Generator().manual_seed(1))
    again = lora.add(y[turned].to(DEV), x[turned].to(DEV), lora.plan(ids[turned].to(DEV)))
    assert torch.equal(again.cpu(), whole.cpu()[turned])


def test_the_projections_of_a_step_share_a_plan_eager_and_in_a_graph():
    """Two BlockLinears with adapters, the plan made in the captured part: replays follow the ids."""
    T, K, N, L = 70, 384, 256, 5
    q, sc, w = fp8_weights(N, K, 1)
    q2, sc2, _ = fp8_weights(K, N, 2)
    up, down = BlockLinear(q.to(DEV), sc.to(DEV)), BlockLinear(q2.to(DEV), sc2.to(DEV))
    a, b, s = C.adapters(L, 16, K, N, 3)
    a2, b2, s2 = C.adapters(L, 8, N, K, 4)
    one, two = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV)), LowRankAdapters(a2.to(DEV), b2.to(DEV), s2.to(DEV))
    x = batch(T, K, N, 5)[0].to(DEV)
    ids = ids_of(T, L, 3, 6).to(DEV)

    def step():
        plan = make_plan(ids, L)
        h = up.forward(x, adapters=one, plan=plan)
        return h, down.forward(h, adapters=two, plan=plan)

    h, y = step()
    base = up.forward(x)
    want, bound = C.add(base, x, a, b, s, ids)
    assert_within(h, want, bound)
    want, bound = C.add(down.forward(h), h, a2, b2, s2, ids)
    assert_within(y, want, bound)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    assert torch.equal(other[0], h) and torch.equal(other[1], y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        if n:
            x.normal_()
            ids.copy_(ids_of(T, L, n, 10 + n))
        h, y = step()
        for v in held:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], h) and torch.equal(held[1], y)


def test_refusals():
    a, b, s = (v.to(DEV) for v in C.adapters(3, 8, 64, 32, 1))
    for args in [(a, b[:, :, :4].contiguous()), (a.half(), b.half()), (a, b.float()), (a, b, s[:2]), (a, b, s.double()), (a[0], b[0]),
                 (a, b.transpose(1, 2)), (torch.zeros(1, 129, 8, device=DEV), torch.zeros(1, 8, 129, device=DEV))]:
        with pytest.raises(ValueError):
            LowRankAdapters(*args)
    lora = LowRankAdapters(a, b, s)
    ids = torch.zeros(5, dtype=torch.int32, device=DEV)
    plan = lora.plan(ids)
    x, y = torch.zeros(5, 64, dtype=BF, device=DEV), torch.zeros(5, 32, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        lora.plan(ids.long())
    for args in [(y, x[:4], plan), (y[:4], x, plan), (y.float(), x, plan), (y, x.half(), plan), (y, x, make_plan(ids, 4)), (y, x, plan, y.float()),
                 (y, x, plan, torch.zeros(5, 64, dtype=BF, device=DEV)[:, ::2])]:
        with pytest.raises(ValueError):
            lora.add(*args)
    with pytest.raises(RuntimeError, match="in its place"):
        wide = torch.zeros(5, 40, dtype=BF, device=DEV)
        lora.add(wide[:, :32], x, plan, wide[:, 4:36])
    q, sc, _ = fp8_weights(32, 128, 1)
    proj = BlockLinear(q.to(DEV), sc.to(DEV))
    with pytest.raises(ValueError):
        proj.forward(torch.zeros(5, 128, dtype=BF, device=DEV), adapters=lora, plan=plan)
    # a plan of another batch writes nothing
    lora.add(y, x, plan._replace(data=lora.plan(ids[:3].contiguous()).data), y)
    assert not y.any()
