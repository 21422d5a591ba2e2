"""netra_moe.norm on the GPU against its 64-bit forms (norm_case.py)."""
import pytest
import torch

import norm_case as N
from conftest import gpu_available
from layers_case import assert_within, blocks
from netra_moe.norm import rms_norm, rms_norm_gradients

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]
BF, F = torch.bfloat16, torch.float32
DEV = "cuda:0"
# one value, odd ends, each number of waves a row and its borders, more rows than workgroups
SIZES = [(1, 1), (1, 7), (2, 8), (3, 128), (5, 130), (4, 511), (6, 512), (5, 513), (7, 1023), (17, 1024), (3, 1025), (9, 1111),
         (1, 2048), (33, 2048), (3, 2049), (2, 4095), (5, 4096), (2, 4097), (3, 8192), (2, 8193), (2, 11111), (3, 16384),
         (9001, 65), (2500, 1030), (70000, 520)]


def tensors(T, H, seed, *dtypes, std=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for dt in dtypes:
        v = torch.randn(T, H, generator=g) * std
        v[:, 3::37] *= 25.0
        out.append(v.to(dt))
    w = (torch.randn(H, generator=g) * 0.3 + 1.0)
    return out, w


def check(n, x, residual, w, codes, eps=1e-6, offset=0.0):
    r = N.normalised(x, residual)
    T, H = r.shape
    if residual is not None:
        assert torch.equal(n.residual.cpu(), r)
    want = N.norm(r, w, eps, offset)
    if n.y is not None:
        N.check_y(n.y, want)
    if codes == "rows":
        N.check_codes(n.codes.cpu().double(), n.scale.cpu(), want)
    elif codes == "tiles":
        N.check_codes(*N.untile(n.codes, n.scale, T, H), want)


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("types", [(BF, BF), (F, None), (BF, F), (F, BF)])
def test_forward(T, H, types):
    (x, *rest), w = tensors(T, H, T + H, *[t for t in types if t])
    residual = rest[0] if rest else None
    w = w.to(BF if H % 2 else F)
    codes = ("rows", "tiles")[(T + H) % 2]
    n = rms_norm(x.to(DEV), w.to(DEV), residual=residual.to(DEV) if rest else None, codes=codes, offset=0.5,
                 out_type=(BF, F)[H % 3 == 0])
    check(n, x, residual, w, codes, offset=0.5)


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("types", [(BF, BF, True), (BF, F, True), (F, F, False), (F, BF, True)])
def test_gradients(T, H, types):
    (dy, r, flow), w = tensors(T, H, 2 * T + H, types[0], types[1], types[1])
    w = w.to(F if H % 2 else BF)
    flow = flow if types[2] else None
    dx, dw = rms_norm_gradients(dy.to(DEV), r.to(DEV), w.to(DEV), residual_gradient=flow.to(DEV) if types[2] else None, offset=-0.25)
    want, want_w, bound, bound_w = N.gradients(dy, r, w, flow, offset=-0.25)
    assert_within(dx, want, bound, "dx")
    assert_within(dw, want_w, bound_w, "dw")
    before = dw.clone()
    rms_norm_gradients(dy.to(DEV), r.to(DEV), w.to(DEV), offset=-0.25, dw=dw, accumulate=True)
    assert torch.equal(dw, before + before)


@pytest.mark.parametrize("codes", ["rows", "tiles", None])
def test_outputs_alone_and_no_rows(codes):
    (x,), w = tensors(19, 260, 4, BF)
    x, w = x.to(DEV), w.to(DEV)
    if codes:
        n = rms_norm(x, w, codes=codes, out_type=None)
        assert n.y is None and n.residual is x
        check(n, x, None, w, codes)
    else:
        n = rms_norm(x, w, out_type=None, residual=x)  # the sum alone
        assert torch.equal(n.residual, x + x)
    e = rms_norm(x[:0], w, codes=codes)
    assert e.y.shape == (0, 260)
    dx, dw = rms_norm_gradients(x[:0], x[:0], w)
    assert dx.shape == (0, 260) and not dw.any()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("H,pad,shift", [(129, 7, 1), (1000, 3, 5), (2047, 1, 3), (4096, 9, 1), (8191, 2, 7)])
def test_strides_alignment_and_neighbours(dtype, H, pad, shift):
    """Column slices at any element offset; what lies beside the rows stays as it was."""
    T, wide = 21, H + pad + shift
    g = torch.Generator().manual_seed(H)
    base = [torch.randn(T, wide, generator=g).to(dtype).to(DEV) for _ in range(4)]
    x, res, out, sums = (b[:, shift:shift + H] for b in base)
    w = torch.randn(H, generator=g).to(DEV)
    kept = [b.clone() for b in base]
    n = rms_norm(x, w, residual=res, out=out, residual_out=sums, codes="rows")
    check(n, x, res, w, "rows")
    for b, k in zip(base[2:], kept[2:]):
        assert torch.equal(b[:, :shift], k[:, :shift]) and torch.equal(b[:, shift + H:], k[:, shift + H:])
    assert torch.equal(base[0], kept[0]) and torch.equal(base[1], kept[1])
    dx, dw = rms_norm_gradients(res, x, w, residual_gradient=sums, out=out)
    want, want_w, bound, bound_w = N.gradients(res, x, w, sums)
    assert_within(dx, want, bound, "dx")
    assert_within(dw, want_w, bound_w, "dw")
    assert torch.equal(base[2][:, :shift], kept[2][:, :shift]) and torch.equal(base[2][:, shift + H:], kept[2][:, shift + H:])


@pytest.mark.parametrize("T,H", [(3, 300), (5000, 700), (700, 4096)])
def test_in_place(T, H):
    (x, res), w = tensors(T, H, 8, BF, BF)
    xd, rd, w = x.to(DEV), res.to(DEV), w.to(DEV)
    n = rms_norm(xd, w, residual=rd, residual_out=rd, out=xd)
    assert n.y is xd and n.residual is rd
    check(n, x, res, w, None)
    dy, flow = x.to(DEV), res.to(DEV)
    want, _, bound, _ = N.gradients(dy, rd, w, flow)
    rms_norm_gradients(dy, rd, w, residual_gradient=flow, out=flow)
    assert_within(flow, want, bound, "dx")


def test_rows_of_zeros_infinities_and_nan_keep_to_themselves():
    (x,), w = tensors(40, 384, 5, F)
    x[3] = 0.0
    x[7, 200] = torch.inf
    x[11, 5] = torch.nan
    x[20] = 1e-30
    n = rms_norm(x.to(DEV), w.to(DEV), codes="rows", out_type=F)
    check(n, x, None, w, "rows")
    assert not n.y[3].any() and torch.isnan(n.y[11]).all() and torch.isnan(n.scale[11]).all()
    assert torch.isnan(n.y[7, 200]) and torch.isfinite(n.y[7, :200]).all()
    assert torch.isnan(n.scale[7, 1]) and torch.isfinite(n.scale[7, [0, 2]]).all()
    zero = rms_norm(torch.zeros(2, 100, device=DEV), w[:100].to(DEV), eps=0.0, codes="tiles")
    assert torch.isnan(zero.y).all()  # 0 / 0


def test_gradient_against_differences():
    """dL/dh along a random direction from two forward passes in fp32: central differences are off by
    h^2 of the third derivative and by 2 * 30 u sum|dy y| / 2h."""
    T, H, h = 6, 520, 1e-2
    g = torch.Generator().manual_seed(9)
    x, d, dy = (torch.randn(T, H, generator=g) for _ in range(3))
    w = torch.randn(H, generator=g)
    f = lambda v: (rms_norm(v.to(DEV), w.to(DEV), out_type=F).y.cpu().double() * dy.double()).sum()  # noqa: E731
    up, down = (x + h * d), (x - h * d)
    dx, _ = rms_norm_gradients(dy.to(DEV), x.to(DEV), w.to(DEV))
    slope = (dx.cpu().double() * (up.double() - down.double())).sum()
    y = N.norm(x, w)
    # a direction of the row's own size turns it by the angle h: the third derivative is at most about 20 |dy y|
    limit = 60 * N.U * (dy.double() * y).abs().sum() + 20 * h ** 3 * (dy.double() * y).norm(dim=1).sum() * H ** 0.5
    assert abs((f(up) - f(down)) - slope) <= limit


def test_another_stream_and_a_captured_graph():
    (x, res, dy), w = tensors(150, 1500, 6, BF, BF, BF)
    x, res, dy, w = (v.to(DEV) for v in (x, res, dy, w))
    want = rms_norm(x, w, residual=res, codes="tiles")
    want_g = rms_norm_gradients(dy, want.residual, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        n = rms_norm(x, w, residual=res, codes="tiles")
        g = rms_norm_gradients(dy, n.residual, w)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gn = rms_norm(x, w, residual=res, codes="tiles")
        gg = rms_norm_gradients(dy, gn.residual, w)
    for k in range(4):
        if k:
            x.copy_(torch.randn_like(x))
            want = rms_norm(x, w, residual=res, codes="tiles")
            want_g = rms_norm_gradients(dy, want.residual, w)
        gn.y.zero_(), gg[1].zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((gn.y, gn.residual, gn.codes, gn.scale, *gg), (want.y, want.residual, want.codes, want.scale, *want_g)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                               b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
        if k == 0:
            for a, b in zip((n.y, n.residual, n.codes, n.scale, *g), (want.y, want.residual, want.codes, want.scale, *want_g)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("change", [dict(weight=torch.ones(8)), dict(weight="short"), dict(residual="shape"), dict(codes="columns"),
                                    dict(out_type=torch.float16), dict(out="strided"), dict(residual_out="x"), dict(eps=-1.0)])
def test_refusals(change):
    x = torch.zeros(3, 16, device=DEV, dtype=BF)
    args = dict(weight=torch.ones(16, device=DEV))
    args.update(change)
    named = {"short": torch.ones(15, device=DEV), "shape": torch.zeros(3, 15, device=DEV), "strided": torch.zeros(3, 32, device=DEV)[:, ::2],
             "x": x}
    args = {k: named.get(v, v) if isinstance(v, str) else v for k, v in args.items()}
    with pytest.raises((ValueError, RuntimeError)):
        rms_norm(x, args.pop("weight"), **args)
