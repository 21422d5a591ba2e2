"""libnetra_layers.so without a GPU: its symbols, workspace sizes and refusals
(every refusal comes before any launch, so made-up pointers are never followed),
and the bounds and formulas of layers_case.py."""
import ctypes

import numpy as np
import pytest
import torch

import layers_case as C
from netra_moe import layers, paths

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")

A = 0x100000000000  # aligned addresses, far apart, that are never followed
B, D = 2 * A, 3 * A


def refused(name, *args):
    lib = layers.library()
    assert getattr(lib, name)(*args) == -1
    text = lib.netra_layers_last_error().decode()
    assert text.startswith(name + ": ") and len(text) > len(name) + 10
    return text


def test_header_declares_every_bound_symbol():
    text = (paths.REPO_ROOT / "include" / "netra_layers.h").read_text()
    for name in layers.SIGNATURES:
        assert f" {name}(" in text or f"*{name}(" in text, name
        assert hasattr(layers.library(), name)


def test_packed_bytes():
    lib = layers.library()
    assert lib.netra_linear_packed_bytes(576, 2048, 0) == 576 * 2048
    assert lib.netra_linear_packed_bytes(5, 7, 0) == 16 * 128
    assert lib.netra_linear_packed_bytes(5, 300, 1) == 304 * 128


@pytest.mark.parametrize("change", [
    dict(x=0), dict(x=A + 1), dict(xt=2), dict(xs=255), dict(packed=0), dict(packed=A + 8), dict(scale=0),
    dict(scale=A + 2), dict(y=0), dict(y=B + 1), dict(ys=127), dict(y=A + 256), dict(y=A + 512 * 299 + 510), dict(y=A - 2), dict(n=0), dict(k=0), dict(rows=(1 << 21) + 1),
    dict(n=(1 << 21) + 1), dict(ws=0), dict(ws=A + 4), dict(wb=0), dict(wb=-1)])
@pytest.mark.parametrize("name", ["netra_linear_forward", "netra_linear_input_gradient"])
def test_product_refusals(name, change):
    lib = layers.library()
    a = dict(x=A, xt=0, xs=256, packed=A, scale=A, y=B, ys=128, rows=300, n=128, k=256, ws=A)
    back = name != "netra_linear_forward"
    if back:
        a.update(n=256, k=128)
    need = getattr(lib, name + "_workspace")(a["rows"], a["n"], a["k"], a["xt"])
    a["wb"] = need
    a.update(change)
    if a["wb"] == -1:
        a["wb"] = need - 1
    refused(name, a["x"], a["xt"], a["xs"], a["packed"], a["scale"], a["y"], a["ys"], a["rows"], a["n"],
            a["k"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("change", [dict(g=0), dict(gt=2), dict(gs=127), dict(x=0), dict(x=A + 1), dict(xt=9), dict(xs=255),
                                    dict(dw=0), dict(dw=D + 2), dict(dw=A), dict(dw=B - 4), dict(dw=B + 300 * 1024 - 4), dict(n=0), dict(k=0), dict(rows=(1 << 21) + 1),
                                    dict(ws=0), dict(ws=A + 8), dict(short=1)])
def test_weight_gradient_refusals(change):
    lib = layers.library()
    # (fp32: both operands go through the workspace)
    a = dict(g=A, gt=1, gs=128, x=B, xt=1, xs=256, dw=D, rows=300, n=128, k=256, ws=A, short=0)
    need = lib.netra_linear_weight_gradient_workspace(300, 128, 256, 0)
    a.update(change)
    refused("netra_linear_weight_gradient", a["g"], a["gt"], a["gs"], a["x"], a["xt"], a["xs"], a["dw"], 0, a["rows"],
            a["n"], a["k"], a["ws"], need - a["short"], None)


@pytest.mark.parametrize("change", [dict(w=0), dict(p=0), dict(p=A), dict(p=2 * A + 8), dict(n=0), dict(k=0),
                                    dict(n=(1 << 21) + 1)])
def test_pack_refusals(change):
    a = dict(w=A, p=2 * A, n=128, k=256)
    a.update(change)
    refused("netra_linear_pack", a["w"], a["p"], a["n"], a["k"], 0, None)


@pytest.mark.parametrize("change", [dict(ids=0), dict(ids=A + 2), dict(st=1), dict(slots=0), dict(E=0), dict(E=1025),
                                    dict(T=1 << 31), dict(T=1 << 30, slots=2), dict(counts=0), dict(counts=A + 1),
                                    dict(ws=A + 4)])
def test_counts_refusals(change):
    a = dict(ids=A, st=2, T=40000, slots=2, E=16, counts=A, ws=A)
    a.update(change)
    if "slots" in change and change["slots"] == 2:
        a["st"] = 2
    if change == dict(ws=A + 4) and not layers.library().netra_router_counts_workspace(a["T"], a["slots"], a["E"]):
        pytest.skip("needs no workspace at this size")
    refused("netra_router_counts", a["ids"], a["st"], None, a["T"], a["slots"], a["E"], a["counts"], 0, a["ws"], 1 << 40,
            None)


@pytest.mark.parametrize("change", [dict(z=0), dict(z=A + 1), dict(zt=2), dict(zs=15), dict(bias=A + 1), dict(ids=0),
                                    dict(ids=A + 2), dict(st=1), dict(E=0), dict(E=1025), dict(T=1 << 31),
                                    dict(counts=0), dict(counts=A + 2), dict(loss=0), dict(loss=A + 1), dict(g=B + 1), dict(g=A), dict(g=A + 2), dict(zs=40, gs=40, g=A + 24),
                                    dict(gs=15), dict(ws=0), dict(ws=A + 4), dict(short=1),
                                    dict(zs=1 << 27), dict(gs=1 << 27)])
def test_balance_refusals(change):
    a = dict(z=A, zt=0, zs=16, bias=None, ids=A, st=2, T=4000, slots=2, E=16, counts=A, loss=A, g=B, gs=16, ws=A, short=0)
    a.update(change)
    need = layers.library().netra_router_balance_workspace(4000, 2, 16)
    refused("netra_router_balance", a["z"], a["zt"], a["zs"], a["bias"], a["ids"], a["st"], a["slots"], None, a["T"],
            a["E"], ctypes.c_float(1.0), a["counts"], a["loss"], a["g"], a["gs"], a["ws"], need - a["short"], None)


def test_quantised_matches_the_layer_oracle(oracle_mod):
    """The 64-bit tests' quantiser against the MoE layer's oracle."""
    x = C.activations(8, 512, seed=3)
    q, s = oracle_mod.quant_rows_bf16(x.view(torch.int16).numpy().view(np.uint16))
    codes = torch.from_numpy(q).view(torch.float8_e4m3fn).double()
    want = (codes.view(8, 4, 128) * torch.from_numpy(s).double()[:, :, None]).view(8, 512)
    assert torch.equal(C.quantised(x, 1), want)


def test_bound_sees_a_wrong_block_scale():
    """The bounds are tight enough: one block's scale off by a fiftieth is outside them."""
    x, (_, _, w) = C.activations(40, 512, seed=5), C.weights(64, 512, seed=6)
    want, bound = C.product(C.quantised(x, 1), w)
    wrong = w.clone()
    wrong[:, 128:256] *= 1.02
    with pytest.raises(AssertionError):
        C.assert_within((C.quantised(x, 1) @ wrong.t()).to(torch.bfloat16), want, bound)
    C.assert_within(want.to(torch.bfloat16), want, bound)


def test_balance_formula_against_autograd():
    g = torch.Generator().manual_seed(3)
    z = torch.randn(9, 12, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, 12, (9, 2), generator=g)
    c = C.counts(ids, 12)
    f = torch.from_numpy(c).double() * 12 / int(c.sum())
    loss = 0.5 * (f * torch.softmax(z, 1).mean(0)).sum()
    loss.backward()
    got = C.balance(z, c, coefficient=0.5)
    assert abs(got[0] - float(loss.detach())) < 1e-15 and torch.allclose(got[1], z.grad, rtol=1e-13, atol=1e-16)
