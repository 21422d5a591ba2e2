"""Every kernel form of the linear layer on the GPU (the sizes of layers_forms.py,
which tests/test_layers_plan.py holds to the forms they are listed for), against
float64 products within the bounds that layers_case.py derives."""
import pytest
import torch

import layers_case as C
import layers_forms as F
from conftest import gpu_available
from netra_moe.linear import BlockLinear

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DEV = torch.device("cuda", 0)
PRODUCTS = [(dt, form, size) for dt, forms in ((torch.bfloat16, F.BF16), (torch.float32, F.F32))
            for form, size in forms.items()]


def layer(n, k, seed, gradients=False):
    q, s, deq = C.weights(n, k, seed)
    return BlockLinear(q.to(DEV), s.to(DEV), gradients=gradients), deq


@pytest.mark.parametrize("direction", ["forward", "input_gradient"])
@pytest.mark.parametrize("dt,form,size", PRODUCTS, ids=lambda v: "-".join(map(str, v)) if isinstance(v, tuple) else None)
def test_product_form(dt, form, size, direction):
    rows, ni, nc = size
    x = C.activations(rows, nc, seed=rows, dtype=dt)
    if direction == "forward":
        lin, w = layer(ni, nc, seed=rows + ni)
        got = lin.forward(x.to(DEV))
    else:
        lin, w = layer(nc, ni, seed=rows + ni, gradients=True)
        got = lin.input_gradient(x.to(DEV))
        w = w.t().contiguous()
    C.assert_within(got, *C.product(C.quantised(x, 1), w))


@pytest.mark.parametrize("size", [s for sizes in F.OUTER.values() for s in sizes], ids=lambda s: "-".join(map(str, s)))
def test_weight_gradient_form(size):
    rows, n, k = size
    lin, _ = layer(n, k, seed=1)
    x, dy = C.activations(rows, k, seed=rows), C.activations(rows, n, seed=rows + 1, std=1e-3)
    dw = lin.weight_gradient(dy.to(DEV), x.to(DEV))
    C.assert_within(dw, *C.outer(dy, x))
    acc = dw.clone()
    lin.weight_gradient(dy.to(DEV), x.to(DEV), acc, accumulate=True)
    assert torch.equal(acc, dw + dw)


@pytest.mark.parametrize("size", F.BACKWARD_IN_ONE + F.BACKWARD_APART, ids=lambda s: "-".join(map(str, s)))
def test_backward_form(size):
    """Both gradients in one launch or apart: the bits of the single calls (a 128-block's
    sums do not depend on the tile)."""
    rows, n, k = size
    lin, w = layer(n, k, seed=2, gradients=True)
    x, dy = C.activations(rows, k, seed=rows), C.activations(rows, n, seed=rows + 1, std=1e-3)
    dx, dw = lin.backward(dy.to(DEV), x.to(DEV))
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")
    assert torch.equal(dx, lin.input_gradient(dy.to(DEV))) and torch.equal(dw, lin.weight_gradient(dy.to(DEV), x.to(DEV)))


def test_copies_that_loop_over_the_rows():
    """Operands too wide for a workgroup per four rows of the copy; whole numbers, so exact."""
    rows, n, k = 7700, 3, 70001
    assert (rows + 3) // 4 > (1 << 18) // -(-k // 512)
    lin = BlockLinear(torch.zeros(n, k, dtype=torch.uint8, device=DEV), torch.ones(1, -(-k // 128), device=DEV))
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randint(-7, 8, (rows, k), generator=g, device=DEV).float()
    dy = torch.randint(-7, 8, (rows, n), generator=g, device=DEV).float()
    assert torch.equal(lin.weight_gradient(dy, x).double(), dy.double().t().contiguous() @ x.double())


@pytest.mark.parametrize("direction", ["forward", "input_gradient"])
@pytest.mark.parametrize("dt,form,size", PRODUCTS, ids=lambda v: "-".join(map(str, v)) if isinstance(v, tuple) else None)
def test_a_row_has_the_same_bits_wherever_it_stands(dt, form, size, direction):
    rows, ni, nc = size
    lin, _ = layer(*((ni, nc) if direction == "forward" else (nc, ni)), seed=3, gradients=direction != "forward")
    x = C.activations(rows, nc, seed=4, dtype=dt).to(DEV)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(5)).to(DEV)
    call = getattr(lin, direction)
    assert torch.equal(call(x[order]), call(x)[order])
