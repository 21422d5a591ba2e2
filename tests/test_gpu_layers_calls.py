"""Calls of the operators beside the layer that their documentation allows: operands
read in place from any four-byte boundary, calls from several threads, graphs that
replay next to each other."""
import threading

import pytest
import torch

import layers_case as C
from conftest import gpu_available
from netra_moe import balance as B
from netra_moe.linear import BlockLinear

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DEV = torch.device("cuda", 0)


def layer(n, k, seed):
    q, s, deq = C.weights(n, k, seed)
    return BlockLinear(q.to(DEV), s.to(DEV), gradients=True), deq


@pytest.mark.parametrize("T", [1, 63, 65, 130, 700])
@pytest.mark.parametrize("offset,pad", [(2, 0), (2, 4), (6, 2), (10, 16)])
def test_operands_in_place_at_four_byte_boundaries(T, offset, pad):
    n, k = 250, 334
    lin, w = layer(n, k, seed=1)
    x, dy = C.activations(T, k, seed=2), C.activations(T, n, seed=3)

    def view(t):  # columns of a wider matrix whose other columns are NaN
        base = torch.full((T, offset + t.shape[1] + pad), torch.nan, dtype=t.dtype, device=DEV)
        base[:, offset:offset + t.shape[1]] = t.to(DEV)
        return base[:, offset:offset + t.shape[1]]

    xv, dyv = view(x), view(dy)
    dx, dw = lin.backward(dyv, xv)
    C.assert_within(lin.forward(xv), *C.product(C.quantised(x, 1), w))
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")
    assert torch.equal(dw, lin.weight_gradient(dyv, xv))


def test_calls_from_several_threads():
    lin, _ = layer(512, 640, seed=4)
    sets = []
    for i, T in enumerate((3, 64, 200, 700)):
        g = torch.Generator().manual_seed(i)
        sets.append((C.activations(T, 640, seed=i).to(DEV), C.activations(T, 512, seed=10 + i).to(DEV),
                     torch.randn(T, 96, generator=g).to(DEV),
                     torch.randint(0, 96, (T, 4), generator=g, dtype=torch.int32).to(DEV)))

    def run(x, dy, z, ids):
        r = B.balance_loss(z, ids)
        return [lin.forward(x), *lin.backward(dy, x), B.expert_counts(ids, 96), r.loss, r.grad]

    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            for _ in range(10):
                got[i].append(run(*sets[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert len(runs) == 10
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_two_graphs_replay_at_once():
    lin, _ = layer(384, 512, seed=5)
    graphs = []
    for i, T in enumerate((300, 900)):
        x, dy = C.activations(T, 512, seed=20 + i).to(DEV), C.activations(T, 384, seed=30 + i).to(DEV)
        z = torch.randn(T, 64, device=DEV)
        ids = torch.randint(0, 64, (T, 2), device=DEV, dtype=torch.int32)
        r = B.balance_loss(z, ids)
        eager = [lin.forward(x), *lin.backward(dy, x), r.loss, r.grad]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = B.balance_loss(z, ids)
            out = [lin.forward(x), *lin.backward(dy, x), r.loss, r.grad]
        graphs.append((graph, torch.cuda.Stream(DEV), out, eager, (x, dy, z, ids)))
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
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
