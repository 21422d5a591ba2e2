"""The norm without a GPU: refusals (before any launch), sizes, its plan and the 64-bit forms' gradients."""
import ctypes

import pytest
import torch

import norm_case as N
from netra_moe import layers, norm, paths
from test_layers_host import A, B, D, refused

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")
F = ctypes.c_float
E = 4 * A


@pytest.mark.parametrize("change", [
    dict(x=0), dict(x=A + 1), dict(xt=2), dict(xs=255), dict(r=B + 1), dict(rt=2), dict(rs=255), dict(r=0), dict(s=0),
    dict(s=D + 1), dict(ss=255), dict(w=0), dict(w=A + 1), dict(wt=5), dict(eps=-1.0), dict(eps=float("nan")), dict(y=E + 1),
    dict(yt=2), dict(ys=255), dict(q=0), dict(qs=0), dict(qs=7 * A + 2), dict(layout=0), dict(layout=3),
    dict(layout=2, q=6 * A + 8), dict(cols=0), dict(cols=16385, xs=20000, rs=20000, ss=20000, ys=20000),
    dict(rows=(1 << 21) + 1), dict(y=A + 2), dict(y=A + 512), dict(s=A + 512), dict(s=E), dict(q=A + 5), dict(qs=5 * A),
    dict(q=E), dict(y=0, q=0, qs=0, r=0, s=0), dict(ss=300, s=B), dict(y=B, ys=300), dict(yt=1, ys=256, y=A)])
def test_forward_refusals(change):
    a = dict(x=A, xt=0, xs=256, r=B, rt=0, rs=256, w=5 * A, wt=0, offset=0.0, eps=1e-6, s=D, ss=256, y=E, yt=0, ys=256,
             q=6 * A, qs=7 * A, layout=1, rows=40, cols=256)
    a.update(change)
    refused("netra_norm_forward", a["x"], a["xt"], a["xs"], a["r"], a["rt"], a["rs"], a["w"], a["wt"], F(a["offset"]),
            F(a["eps"]), a["s"], a["ss"], a["y"], a["yt"], a["ys"], a["q"], a["qs"], a["layout"], a["rows"], a["cols"], None)


@pytest.mark.parametrize("change", [
    dict(g=0), dict(g=A + 1), dict(gt=2), dict(gs=255), dict(r=0), dict(r=B + 1), dict(rt=3), dict(rs=255), dict(f=D + 1),
    dict(fs=255), dict(w=0), dict(wt=2), dict(o=0), dict(o=E + 1), dict(os=255), dict(dw=0), dict(dw=6 * A + 2), dict(dw=A),
    dict(dw=5 * A), dict(dw=E + 4), dict(o=A + 512), dict(o=5 * A), dict(gt=1, o=A), dict(os=300, o=B), dict(eps=-1.0),
    dict(cols=0), dict(cols=16385, gs=20000, rs=20000, fs=20000, os=20000), dict(rows=(1 << 21) + 1), dict(ws=0), dict(ws=7 * A + 8),
    dict(short=1)])
def test_gradient_refusals(change):
    a = dict(g=A, gt=0, gs=256, r=B, rt=0, rs=256, f=D, fs=256, w=5 * A, wt=0, eps=1e-6, o=E, os=256, dw=6 * A, rows=40,
             cols=256, ws=7 * A, short=0)
    need = layers.library().netra_norm_gradients_workspace(40, 256)
    a.update(change)
    refused("netra_norm_gradients", a["g"], a["gt"], a["gs"], a["r"], a["rt"], a["rs"], a["f"], a["fs"], a["w"], a["wt"],
            F(0.0), F(a["eps"]), a["o"], a["os"], a["dw"], 0, a["rows"], a["cols"], a["ws"], need - a["short"], None)


def test_sizes():
    lib = layers.library()
    assert lib.netra_norm_code_bytes(5, 300, 1) == 1500 and lib.netra_norm_scale_count(5, 300, 1) == 15
    assert lib.netra_norm_code_bytes(5, 300, 2) == 16 * 384 and lib.netra_norm_scale_count(17, 300, 2) == 32 * 3
    assert lib.netra_norm_gradients_workspace(0, 256) == 0


def test_no_rows_launch_nothing():
    lib = layers.library()
    assert lib.netra_norm_forward(A, 0, 8, None, 0, 0, B, 0, F(0), F(0), None, 0, D, 0, 8, None, None, 0, 0, 8, None) == 0
    assert lib.netra_norm_gradients(None, 0, 0, None, 0, 0, None, 0, A, 0, F(0), F(0), None, 0, B, 1, 0, 8, None, 0, None) == 0


@pytest.mark.parametrize("call", [
    lambda: norm.rms_norm(torch.zeros(2, 4), torch.zeros(4)),
    lambda: norm.rms_norm_gradients(torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(4))])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="GPU tensor"):
        call()


def test_gradient_formula_against_autograd_and_differences():
    g = torch.Generator().manual_seed(1)
    r = torch.randn(5, 9, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(9, generator=g, dtype=torch.float32).double().requires_grad_()
    dy, flow = torch.randn(5, 9, generator=g, dtype=torch.float64), torch.randn(5, 9, generator=g, dtype=torch.float64)

    def loss(r, w):
        return ((r / (r.square().mean(1, keepdim=True) + 1e-6).sqrt() * (w + 1.0)) * dy).sum() + (r * flow).sum()

    dr, dw = torch.autograd.grad(loss(r, w), (r, w))
    got = N.gradients(dy, r.detach(), w.detach(), flow, offset=1.0)
    assert torch.allclose(got[0], dr, rtol=1e-12, atol=1e-12) and torch.allclose(got[1], dw, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(loss, (r, w))
    assert torch.allclose(N.norm(r.detach(), w.detach(), offset=1.0) * 1.0, r.detach() / (r.detach().square().mean(1, keepdim=True) + 1e-6).sqrt() * (w.detach() + 1.0))


def test_untile_inverts_the_layout():
    rows, cols = 37, 300
    codes = torch.zeros(48 * 384, dtype=torch.uint8)
    want = torch.randint(0, 120, (48, 384), dtype=torch.uint8)
    for row in range(48):
        for c in range(384):
            b, i = c // 128, c % 128
            codes[((row // 16) * 3 + b) * 2048 + (i % 32) // 16 * 1024 + ((row % 16) + 16 * (i // 32)) * 16 + i % 16] = want[row, c]
    got, _ = N.untile(codes, torch.zeros(3, 48), rows, cols)
    assert torch.equal(got, want.view(torch.float8_e4m3fn).double()[:rows, :cols])


@pytest.mark.parametrize("change", [dict(c=0), dict(c=A + 8), dict(s=0), dict(s=B + 2), dict(p=0), dict(p=D + 8), dict(w=0), dict(w=E + 2),
                                    dict(y=0), dict(y=5 * A + 1), dict(ys=127), dict(n=0), dict(k=0), dict(rows=(1 << 21) + 1), dict(y=A), dict(y=B),
                                    dict(k=8192, ws=0), dict(k=8192, ws=6 * A + 4), dict(k=8192, short=1)])
def test_codes_product_refusals(change):
    a = dict(c=A, s=B, p=D, w=E, y=5 * A, ys=128, rows=300, n=128, k=256, ws=6 * A, short=0)
    a.update(change)
    need = layers.library().netra_linear_forward_codes_workspace(300, 128, a["k"])
    assert bool(need) == (a["k"] == 8192)
    refused("netra_linear_forward_codes", a["c"], a["s"], a["p"], a["w"], a["y"], a["ys"], a["rows"], a["n"], a["k"], a["ws"],
            need - a["short"], None)
