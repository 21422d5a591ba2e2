"""The norm, the routing and the adapters where element offsets pass 32 bits, by row strides (rows of one
allocation, of which only they are written), and of as many rows as their documentation allows."""
import pytest
import torch

import adapters_case as A
import norm_case as N
import routing_case as R
from conftest import gpu_available
from layers_case import assert_within
from netra_moe.adapters import LowRankAdapters
from netra_moe.norm import rms_norm, rms_norm_gradients
from netra_moe.routing import route, route_gradient

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = "cuda:0"


def apart(values, stride):
    """The rows of `values` on the GPU, `stride` elements apart."""
    rows, cols = values.shape
    store = torch.empty((rows - 1) * stride + cols, dtype=values.dtype, device=DEV)
    view = torch.as_strided(store, (rows, cols), (stride, 1))
    view.copy_(values)
    return view


@pytest.mark.parametrize("dtype,stride", [(BF, (1 << 30) + 3), (F, (1 << 29) + 1)])
@pytest.mark.parametrize("H", [300, 5000])
def test_norm_of_rows_far_apart(dtype, stride, H):
    g = torch.Generator().manual_seed(H)
    x, res, dy = (torch.randn(9, H, generator=g).to(dtype) for _ in range(3))
    w = torch.rand(H, generator=g)
    xs, rs = apart(x, stride), apart(res, stride)
    n = rms_norm(xs, w.to(DEV), residual=rs, out_type=F, codes="rows")
    r = N.normalised(x, res)
    N.check_y(n.y, N.norm(r, w))
    assert torch.equal(n.residual.cpu(), r)
    again = rms_norm(xs, w.to(DEV), residual=rs, out=xs, residual_out=rs, codes="rows")  # in place
    assert again.y is xs and torch.equal(rs.cpu(), r) and torch.equal(again.codes.view(torch.uint8), n.codes.view(torch.uint8))
    assert torch.equal(xs, n.y.to(dtype))
    want, dw_want, bound, dw_bound = N.gradients(dy, r, w, r)
    dx, dw = rms_norm_gradients(dy.to(DEV), rs, w.to(DEV), residual_gradient=rs, out=rs)
    assert_within(dx, want, bound, "dx")
    assert_within(dw, dw_want, dw_bound, "dw")


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("E", [64, 600])
def test_routing_of_rows_far_apart(dtype, E):
    """The largest stride, and 33 rows of it: the last begins 2^32 elements on."""
    T, k, stride = 34, 5, (1 << 27) - 1
    z = R.inputs(T, E, E, dtype)
    zs = apart(z, stride)
    bias = (torch.rand(E, generator=torch.Generator().manual_seed(1)) - 0.5) * 0.1
    for kw in (dict(), dict(scoring="sigmoid", selection_bias=bias.to(DEV), groups=4, top_groups=2, group_score="top2")):
        r = route(zs, k, **kw)
        grouped = (bias, 4, 2, "top2") if kw else ()
        ids = R.choose(z, k, kw.get("scoring", "softmax"), *grouped)
        assert torch.equal(r.ids.cpu().long(), ids)
        scoring = kw.get("scoring", "softmax")
        want, bound = R.weights(z, ids, scoring)
        assert_within(r.weights, want, bound, "weights")
        dw = torch.randn(T, k, generator=torch.Generator().manual_seed(2))
        out = torch.as_strided(torch.empty(1, dtype=dtype, device=DEV).resize_((T - 1) * stride + E), (T, E), (stride, 1))
        route_gradient(dw.to(DEV), zs, r.ids, scoring=scoring, out=out)
        want, bound = R.gradient(dw, z, ids, scoring)
        assert_within(out, want, bound, "grad")
        del out


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("r,K,N_", [(8, 100, 130), (70, 9000, 600)])
def test_adapters_of_rows_far_apart(dtype, r, K, N_):
    T, L, stride = 9, 3, (1 << 29) + 1
    g = torch.Generator().manual_seed(r)
    a, b, s = A.adapters(L, r, K, N_, r)
    x, y = torch.randn(T, K, generator=g).to(dtype), torch.randn(T, N_, generator=g).to(BF)
    ids = torch.randint(-1, L, (T,), generator=g, dtype=torch.int32)
    lora = LowRankAdapters(a.to(DEV), b.to(DEV), s.to(DEV))
    ys = apart(y, 2 * stride)
    assert lora.add(ys, apart(x, stride), lora.plan(ids.to(DEV)), ys) is ys
    assert_within(ys, *A.add(y, x, a, b, s, ids))


def test_as_many_rows_as_the_norm_takes():
    T, H = 1 << 21, 40
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = torch.randn(T, H, generator=g, device=DEV).to(BF), torch.rand(H, generator=g, device=DEV)
    n = rms_norm(x, w, out_type=F, codes="tiles")
    dx, dw = rms_norm_gradients(x, x, w)
    codes, scale = n.codes.view(T // 16, -1), n.scale
    for rows in (slice(0, 48), slice(T - 48, T)):
        few = rms_norm(x[rows], w, out_type=F, codes="tiles")
        assert torch.equal(n.y[rows], few.y) and torch.equal(scale[:, rows], few.scale)
        assert torch.equal(codes[rows.start // 16:rows.stop // 16].flatten(), few.codes)
        assert torch.equal(dx[rows], rms_norm_gradients(x[rows], x[rows], w)[0])
    r = x.double()
    terms = r * (r / (r.square().mean(1, keepdim=True) + 1e-6).sqrt())
    assert_within(dw, terms.sum(0).cpu(), ((T + 60) * N.U * terms.abs().sum(0)).cpu(), "dw")


@pytest.mark.parametrize("E", [3, 513])
def test_as_many_tokens_as_the_routing_takes(E):
    """Runs of the same logits: what a call of one run gives, in each place."""
    T, run, k = 1 << 25, 1 << 13, 2
    some = R.inputs(run, E, E, BF).to(DEV)
    z = some.repeat(T // run, 1)
    r = route(z, k, scoring="sigmoid")
    want = route(some, k, scoring="sigmoid")
    assert torch.equal(want.ids.cpu().long(), R.choose(some.cpu(), k))
    for got, of_run in zip(r, want):
        assert bool((got.view(T // run, run, k) == of_run).all())
    dw = torch.randn(run, k, device=DEV)
    grad = route_gradient(dw.repeat(T // run, 1), z, r.ids, scoring="sigmoid", out=torch.empty_like(z))
    of_run = route_gradient(dw, some, want.ids, scoring="sigmoid")
    assert all(bool((part == of_run).all()) for part in grad.view(T // run, run, E).split(64))
