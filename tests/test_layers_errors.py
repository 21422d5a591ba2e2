"""Errors of HIP calls that the layers and weight-prep libraries did not make: an error that an
earlier call left on the thread is the caller's, and a call that runs is not
reported as failed for it."""
import ctypes

import pytest
import torch

import layers_case as C
from conftest import gpu_available
from netra_moe import balance as B
from netra_moe import layers, paths
from netra_moe import weights as W
from netra_moe.linear import BlockLinear

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")

INVALID_DEVICE = 101  # hipErrorInvalidDevice


def hip(name, *args):
    """A HIP runtime call of the library's own runtime."""
    fn = getattr(layers.library(), name)
    fn.restype = ctypes.c_int
    return fn(*args)


def test_a_call_that_launches_nothing_succeeds_whatever_came_before():
    """No tokens and accumulate: nothing to do, with a stale error and without any device."""
    hip("hipSetDevice", 12345)
    lib = layers.library()
    dw = 0x100000000000  # never followed
    assert lib.netra_linear_weight_gradient(None, 0, 4, None, 0, 4, dw, 1, 0, 4, 4, None, 0, None) == 0
    assert lib.netra_layers_last_error() == b""
    hip("hipGetLastError")


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs a GPU")
def test_calls_run_behind_a_stale_error_and_leave_it_to_the_caller():
    dev = torch.device("cuda", 0)
    q, s, w = C.weights(200, 300, seed=1)
    x, dy = C.activations(70, 300, seed=2), C.activations(70, 200, seed=3)
    xd, dyd = x.to(dev), dy.to(dev)
    lin = BlockLinear(q.to(dev), s.to(dev), gradients=True)
    z = torch.randn(300, 16, device=dev)
    ids = torch.randint(0, 16, (300, 2), device=dev, dtype=torch.int32)
    outs = (torch.empty(70, 200, dtype=torch.bfloat16, device=dev), torch.empty(16, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert hip("hipSetDevice", 12345) == INVALID_DEVICE
    try:
        lin.forward(xd, outs[0])
        dx, dw = lin.backward(dyd, xd)
        B.expert_counts(ids, 16, out=outs[1])
        r = B.balance_loss(z, ids)
        assert hip("hipPeekAtLastError") == INVALID_DEVICE
    finally:
        hip("hipGetLastError")
    assert hip("hipPeekAtLastError") == 0
    C.assert_within(outs[0], *C.product(C.quantised(x, 1), w))
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")
    want = C.counts(ids, 16)
    assert outs[1].tolist() == want.tolist() == r.counts.tolist()
    assert torch.isfinite(r.loss) and torch.isfinite(r.grad).all()


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs a GPU")
def test_weight_prep_runs_behind_a_stale_error():
    w = torch.randn(2, 128, 256, device="cuda:0") * 0.02
    q, s = W.quantize_blocks(w)
    packed = [W.pack_tiles(q), W.pack_tiles(q, gate_up=True), W.pack_tiles_from_aiter(q)]
    torch.cuda.synchronize()
    assert hip("hipSetDevice", 12345) == INVALID_DEVICE
    try:
        again = W.quantize_blocks(w)
        repacked = [W.pack_tiles(q), W.pack_tiles(q, gate_up=True), W.pack_tiles_from_aiter(q)]
        assert hip("hipPeekAtLastError") == INVALID_DEVICE
    finally:
        hip("hipGetLastError")
    assert torch.equal(again[0], q) and torch.equal(again[1], s)
    assert all(torch.equal(a, b) for a, b in zip(packed, repacked))
