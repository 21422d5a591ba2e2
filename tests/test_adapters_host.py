"""The adapters without a GPU: refusals (before any launch), sizes and the bound."""
import pytest
import torch

import adapters_case as C
from netra_moe import adapters, layers, paths
from test_layers_host import A, B, D, refused

pytestmark = pytest.mark.skipif(not paths.layers_library().is_file(), reason="library not built")


@pytest.mark.parametrize("change", [
    dict(x=0), dict(x=A + 1), dict(xt=2), dict(xs=8191), dict(pa=0), dict(pa=B + 8), dict(pb=0), dict(pb=D + 4), dict(scale=0),
    dict(scale=4 * A + 2), dict(plan=0), dict(plan=5 * A + 8), dict(y=0), dict(y=6 * A + 1), dict(ys=127), dict(o=0), dict(o=7 * A + 1),
    dict(os=127), dict(o=A), dict(o=6 * A + 2), dict(os=200, o=6 * A), dict(T=(1 << 21) + 1), dict(L=0), dict(L=1025), dict(r=0),
    dict(r=129), dict(n=0), dict(k=0), dict(n=(1 << 21) + 1, ys=1 << 22, os=1 << 22), dict(ws=0), dict(ws=8 * A + 8), dict(short=1)])  # (of two launches)
def test_add_refusals(change):
    a = dict(x=A, xt=0, xs=8192, pa=B, pb=D, scale=4 * A, plan=5 * A, y=6 * A, ys=128, o=7 * A, os=128, T=40, L=3, r=100, n=128,
             k=8192, ws=8 * A, short=0)
    need = layers.library().netra_adapters_add_workspace(40, 3, 100, 128, 8192)
    a.update(change)
    refused("netra_adapters_add", a["x"], a["xt"], a["xs"], a["pa"], a["pb"], a["scale"], a["plan"], a["y"], a["ys"], a["o"],
            a["os"], a["T"], a["L"], a["r"], a["n"], a["k"], a["ws"], need - a["short"], None)


@pytest.mark.parametrize("change", [dict(a=0), dict(a=A + 1), dict(b=0), dict(b=B + 1), dict(type=2), dict(pa=0), dict(pa=D + 8),
                                    dict(pb=0), dict(pb=4 * A + 8), dict(pa=A), dict(pb=B + 16), dict(pb=D + 16), dict(L=0), dict(L=1025),
                                    dict(r=0), dict(r=129), dict(n=0), dict(k=0)])
def test_pack_refusals(change):
    a = dict(a=A, b=B, type=0, pa=D, pb=4 * A, L=3, r=8, n=128, k=256)
    a.update(change)
    refused("netra_adapters_pack", a["a"], a["b"], a["type"], a["pa"], a["pb"], a["L"], a["r"], a["n"], a["k"], None)


@pytest.mark.parametrize("change", [dict(ids=0), dict(ids=A + 2), dict(T=(1 << 21) + 1), dict(L=0), dict(L=1025), dict(plan=0),
                                    dict(plan=B + 4), dict(plan=A), dict(short=1)])
def test_plan_refusals(change):
    a = dict(ids=A, T=40, L=3, plan=B, short=0)
    need = layers.library().netra_adapters_plan_bytes(40, 3)
    a.update(change)
    refused("netra_adapters_plan", a["ids"], a["T"], a["L"], a["plan"], need - a["short"], None)


def test_sizes_and_no_tokens():
    lib = layers.library()
    assert lib.netra_adapters_packed_bytes(3, 16, 64, 128, 0) == 3 * 16 * 128 * 2
    assert lib.netra_adapters_packed_bytes(3, 17, 65, 129, 0) == 3 * 32 * 256 * 2
    assert lib.netra_adapters_packed_bytes(3, 17, 65, 129, 1) == 3 * 32 * 128 * 2
    assert lib.netra_adapters_plan_bytes(0, 3) == 0 == lib.netra_adapters_add_workspace(0, 3, 8, 8, 8)
    assert lib.netra_adapters_plan(None, 0, 3, None, 0, None) == 0
    assert lib.netra_adapters_add(None, 0, 0, None, None, None, None, None, 0, None, 0, 0, 3, 8, 8, 8, None, 0, None) == 0


def test_most_tiles_of_a_batch():
    """The plan holds the most tiles that any split of the tokens over the adapters (and none) gives."""
    lib = layers.library()
    for T, L in [(1, 1), (2, 5), (40, 3), (63, 64), (1025, 8), (2000, 50), (2000, 63), (8192, 8), (8200, 128), (8200, 129)]:
        tile = 32 if T >= 8192 and T // 64 >= L else 16
        parts = min(L + 1, T)
        most = parts + (T - parts) // tile  # one token each, the rest in one
        assert lib.netra_adapters_plan_bytes(T, L) >= 16 + 4 * T + 16 * most


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        adapters.LowRankAdapters(torch.zeros(1, 2, 4), torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="GPU tensor"):
        adapters.make_plan(torch.zeros(3, dtype=torch.int32), 2)


def test_bound_sees_a_wrong_adapter():
    g = torch.Generator().manual_seed(1)
    a, b, s = C.adapters(3, 8, 200, 50, 2)
    x, y = torch.randn(30, 200, generator=g).to(torch.bfloat16), torch.randn(30, 50, generator=g).to(torch.bfloat16)
    ids = torch.randint(-1, 3, (30,), generator=g)
    want, bound = C.add(y, x, a, b, s, ids)
    C.assert_within(want.to(torch.bfloat16), want, bound)
    wrong, _ = C.add(y, x, a, b, s * 1.05, ids)
    with pytest.raises(AssertionError):
        C.assert_within(wrong.to(torch.bfloat16), want, bound)
