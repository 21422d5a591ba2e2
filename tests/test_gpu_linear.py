"""netra_moe.linear (block-FP8 linear layer and its gradients) on the GPU against
float64 products of the quantised operands, within the bounds layers_case.py
derives."""
import pytest
import torch

import layers_case as C
from conftest import gpu_available
from netra_moe.linear import BlockLinear

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a GPU")]

DEV = torch.device("cuda", 0)
BF16, F32 = torch.bfloat16, torch.float32

# rows around every tile edge, sizes inside and across the 16 / 128 blocks, long contractions
SHAPES = [(1, 128, 128), (1, 2048, 2048), (1, 5, 7), (1, 320, 16384), (2, 130, 257), (5, 576, 512), (15, 16, 128),
          (16, 256, 640), (17, 1000, 333), (33, 129, 2048), (48, 64, 100), (64, 512, 2048), (65, 264, 384),
          (100, 2048, 512), (127, 127, 127), (128, 128, 1024), (130, 1, 300), (200, 3, 1000), (256, 256, 256),
          (257, 513, 1025), (300, 1024, 640), (513, 384, 200), (700, 1030, 520), (1024, 512, 130), (40, 7, 1), (90, 1, 1)]


def layer(n, k, seed, gradients=False):
    q, s, deq = C.weights(n, k, seed)
    return BlockLinear(q.to(DEV), s.to(DEV), gradients=gradients), deq


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_forward(T, N, K, xt):
    lin, w = layer(N, K, seed=T + N + K)
    x = C.activations(T, K, seed=T, dtype=xt)
    y = lin.forward(x.to(DEV))
    assert y.dtype == BF16
    C.assert_within(y, *C.product(C.quantised(x, 1), w))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_gradients(T, N, K, dt):
    lin, w = layer(N, K, seed=T + N + K, gradients=True)
    x, dy = C.activations(T, K, seed=T, dtype=dt), C.activations(T, N, seed=T + 1, dtype=dt, std=1e-3)
    dx, dw = lin.backward(dy.to(DEV), x.to(DEV))
    assert dx.dtype == BF16 and dw.dtype == F32
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")


# sizes that take the largest tiles, with ragged last ones
@pytest.mark.parametrize("T,N,K", [(4095, 4097, 257), (4100, 4000, 100), (1500, 4001, 260)])
def test_forward_of_many_tiles(T, N, K):
    lin, w = layer(N, K, seed=T)
    x = C.activations(T, K, seed=T)
    C.assert_within(lin.forward(x.to(DEV)), *C.product(C.quantised(x, 1), w))


@pytest.mark.parametrize("T,N,K", [(130, 4001, 3999), (70, 4000, 4000), (1300, 2050, 2050)])
def test_weight_gradient_of_many_tiles(T, N, K):
    lin, _ = layer(N, K, seed=T)
    x, dy = C.activations(T, K, seed=T), C.activations(T, N, seed=T + 1, std=1e-3)
    C.assert_within(lin.weight_gradient(dy.to(DEV), x.to(DEV)), *C.outer(dy, x))


def test_weight_gradient_of_mixed_types():
    lin, _ = layer(200, 300, seed=1)
    x, dy = C.activations(150, 300, seed=2, dtype=F32), C.activations(150, 200, seed=3)
    C.assert_within(lin.weight_gradient(dy.to(DEV), x.to(DEV)), *C.outer(dy, x))
    C.assert_within(lin.weight_gradient(dy.to(DEV).float(), x.to(DEV).to(BF16)), *C.outer(dy, x))


def whole(t, n, g, most=7):
    """Whole numbers up to 7 with a 7 in every 128-group: 64 v is their code for a scale of 7/448."""
    v = torch.randint(-most, most + 1, (t, n), generator=g).float()
    v[:, ::128] = 7.0
    return v


@pytest.mark.parametrize("T,N,K", SHAPES)
def test_whole_numbers_are_exact(T, N, K):
    """Codes 64 v and weights of -3 .. 3 lose nothing in the matrix core; a scale of
    1/64 (7/448 rounded to fp32 and back) is off by u or two, so before the rounding
    to bf16 the outputs are within 4 (2 + blocks + splits) u of whole sums."""
    g = torch.Generator().manual_seed(T * N + K)
    w = torch.randint(-3, 4, (N, K), generator=g).float()
    scale = 2.0 ** torch.randint(-1, 2, (C.blocks(N), C.blocks(K)), generator=g).float()
    lin = BlockLinear(w.to(torch.float8_e4m3fn).to(DEV), scale.to(DEV), gradients=True)
    values = (w * scale.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).double()
    x, dy = whole(T, K, g), whole(T, N, g)
    for got, a, b in ((lin.forward(x.to(DEV)), x, values.t()), (lin.input_gradient(dy.to(DEV)), dy, values)):
        a = a.double()
        C.assert_within(got, a @ b, 4 * (2 + C.blocks(a.shape[1]) + C.SPLITS) * C.U * (a.abs() @ b.abs()))
    want = dy.double().t() @ x.double()  # sums below 2^24: exact
    assert torch.equal(lin.weight_gradient(dy.to(DEV), x.to(DEV)).cpu().double(), want)


def test_gradients_are_the_derivatives():
    """For whole numbers that the quantisation keeps, <dy, y(x + d) - y(x)> is <dx, d>
    and <dW, E> is <dy, x E^T>. y and dx are bf16: off by 2^-8 of themselves."""
    g = torch.Generator().manual_seed(0)
    T, N, K = 24, 256, 384
    w = torch.randint(-3, 4, (N, K), generator=g).float()
    lin = BlockLinear(w.to(torch.float8_e4m3fn).to(DEV), torch.ones(2, 3, device=DEV), gradients=True)
    x, dy = whole(T, K, g), whole(T, N, g)
    x2 = (x + torch.randint(-2, 3, (T, K), generator=g)).clamp(-7, 7)
    x2[:, ::128] = 7.0
    y1, y2 = (lin.forward(v.to(DEV)).cpu().double() for v in (x, x2))
    dx, dw = (v.cpu().double() for v in lin.backward(dy.to(DEV), x.to(DEV)))
    lhs, rhs = (dy.double() * (y2 - y1)).sum(1), (dx * (x2 - x).double()).sum(1)
    slack = 1.01 * 2.0 ** -8 * ((dy.abs().double() * (y1.abs() + y2.abs())).sum(1) + (dx.abs() * (x2 - x).abs()).sum(1))
    assert torch.all((lhs - rhs).abs() <= slack) and (lhs.abs() > 2 * slack).sum() >= T // 4
    e = torch.randint(-2, 3, (N, K), generator=g).double()
    assert float((dw * e).sum()) == float((dy.double() * (x.double() @ e.t())).sum())


def test_rows_with_infinities_and_nan_stay_in_their_rows():
    lin, w = layer(160, 400, seed=4, gradients=True)
    x = C.activations(40, 400, seed=5, dtype=F32)
    x[3, 130], x[17, 399], x[20, 0], x[21] = torch.inf, torch.nan, -torch.inf, torch.nan
    y = lin.forward(x.to(DEV))
    want, bound = C.product(C.quantised(x, 1), w)
    assert torch.isnan(want).any(1).sum() == 4 and torch.isnan(want).all(1).sum() == 4
    C.assert_within(y, want, bound)
    dy = C.activations(40, 160, seed=6, dtype=F32)
    C.assert_within(lin.weight_gradient(dy.to(DEV), x.to(DEV)), *C.outer(dy, x))


def test_extreme_magnitudes():
    lin, w = layer(64, 300, seed=7)
    x = torch.zeros(6, 300)
    x[1], x[2], x[3] = 1e-30, 1e37, torch.randn(300) * 1e-12
    x[4, 0], x[5, 299] = 2.0 ** -126, 1.0
    y = lin.forward(x.to(DEV))
    C.assert_within(y, *C.product(C.quantised(x, 1), w))
    assert torch.equal(y[:2].cpu(), torch.zeros(2, 64, dtype=BF16))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("T", [1, 16, 40, 130])
@pytest.mark.parametrize("offset,pad", [(0, 0), (8, 8), (1, 0), (3, 5), (4, 4)])
def test_strides_and_alignments(T, offset, pad, dt):
    """Views with any row stride and offset, in and out; nothing around the output
    is written."""
    N, K = 136, 260
    lin, w = layer(N, K, seed=11, gradients=True)
    x, dy = C.activations(T, K, seed=12, dtype=dt), C.activations(T, N, seed=13, dtype=dt)
    def view(v):
        base = torch.full((T + 2, offset + v.shape[1] + pad), 77.0, dtype=dt, device=DEV)
        base[1:T + 1, offset:offset + v.shape[1]] = v.to(DEV)
        return base[1:T + 1, offset:offset + v.shape[1]]
    xv, dyv = view(x), view(dy)
    base = torch.full((T + 2, offset + N + pad), 55.0, dtype=BF16, device=DEV)
    out = base[1:T + 1, offset:offset + N]
    assert lin.forward(xv, out) is out
    C.assert_within(out, *C.product(C.quantised(x, 1), w))
    around = base.clone()
    around[1:T + 1, offset:offset + N] = 55.0
    assert torch.all(around == 55.0)
    dx, dw = lin.backward(dyv, xv)
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")


@pytest.mark.parametrize("T,N,K", [(64, 256, 512), (300, 130, 257), (2000, 256, 128), (5, 40, 60)])
def test_weight_gradient_accumulates(T, N, K):
    lin, _ = layer(N, K, seed=14)
    x, dy = C.activations(T, K, seed=15).to(DEV), C.activations(T, N, seed=16).to(DEV)
    once = lin.weight_gradient(dy, x)
    acc = torch.full((N, K), 3.0, device=DEV)
    assert lin.weight_gradient(dy, x, acc, accumulate=True) is acc
    assert torch.equal(acc, once + 3.0)
    lin.weight_gradient(dy, x, acc)
    assert torch.equal(acc, once)


def test_no_rows():
    lin, _ = layer(100, 200, seed=17, gradients=True)
    x, dy = torch.empty(0, 200, dtype=BF16, device=DEV), torch.empty(0, 100, dtype=BF16, device=DEV)
    assert lin.forward(x).shape == (0, 100)
    dx, dw = lin.backward(dy, x)
    assert dx.shape == (0, 200) and torch.equal(dw, torch.zeros(100, 200, device=DEV))
    dw += 2.0
    assert torch.equal(lin.weight_gradient(dy, x, dw, accumulate=True), torch.full((100, 200), 2.0, device=DEV))


@pytest.mark.parametrize("T", [1, 8, 40, 500])
def test_repeats_and_batch_position_give_the_same_bits(T):
    lin, _ = layer(384, 640, seed=18, gradients=True)
    x, dy = C.activations(T, 640, seed=19).to(DEV), C.activations(T, 384, seed=20).to(DEV)
    first = (lin.forward(x), *lin.backward(dy, x))
    for _ in range(3):
        for a, b in zip(first, (lin.forward(x), *lin.backward(dy, x))):
            assert torch.equal(a, b)


def test_from_float_and_codes_agree():
    q, s, _ = C.weights(200, 330, seed=21)
    g = torch.Generator().manual_seed(21)
    w = torch.randn(200, 330, generator=g) * 0.02
    x = C.activations(9, 330, seed=22).to(DEV)
    a = BlockLinear.from_float(w.to(DEV)).forward(x)
    b = BlockLinear(q.view(torch.uint8).to(DEV), s.to(DEV)).forward(x)
    assert torch.equal(a, b)


def test_from_checkpoint_with_output_shards_and_bf16_scales():
    q, s, _ = C.weights(576, 320, seed=23)
    s16 = s.to(BF16)
    want = BlockLinear(q.to(DEV), s16.float().to(DEV))
    shards = {"m.o_proj.weight": [q[:256], q[256:]], "m.o_proj.weight_scale_inv": [s16[:2], s16[2:]]}
    got = BlockLinear.from_checkpoint(shards, "m.o_proj", DEV, gradients=True)
    assert torch.equal(got.packed, want.packed) and torch.equal(got.scale, want.scale)
    with pytest.raises(KeyError):
        BlockLinear.from_checkpoint(shards, "m.q_proj", DEV)


def test_captured_graph_replays_beside_eager_work():
    lin, _ = layer(384, 512, seed=24, gradients=True)
    x, dy = C.activations(70, 512, seed=25).to(DEV), C.activations(70, 384, seed=26).to(DEV)
    lin.forward(x), lin.backward(dy, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin.forward(x)
        dx, dw = lin.backward(dy, x)
    for i in range(4):
        x.copy_(C.activations(70, 512, seed=30 + i))
        dy.copy_(C.activations(70, 384, seed=40 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dx, dw), (lin.forward(x), *lin.backward(dy, x))):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    lin, _ = layer(1024, 1024, seed=27, gradients=True)
    xs = [C.activations(t, 1024, seed=28 + t).to(DEV) for t in (300, 7, 64, 1)]
    want = [lin.forward(x) for x in xs]
    grads = [lin.weight_gradient(w, x) for w, x in zip(want, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in xs]
    for _ in range(5):
        got = []
        for st, x, w in zip(streams, xs, want):
            with torch.cuda.stream(st):
                got.append((lin.forward(x), lin.weight_gradient(w, x)))
        torch.cuda.synchronize()
        for (a, b), w, g in zip(got, want, grads):
            assert torch.equal(a, w) and torch.equal(b, g)


def test_refusals():
    lin, _ = layer(128, 256, seed=29)
    x = torch.zeros(4, 256, dtype=BF16, device=DEV)
    for bad in (x.half(), x.t(), x[:, ::2], x[:, :255], x.cpu(), x[0], x.expand(4, 256)[:1].expand(4, 256)):
        with pytest.raises(ValueError):
            lin.forward(bad)
    for out in (torch.empty(4, 128, dtype=F32, device=DEV), torch.empty(3, 128, dtype=BF16, device=DEV)):
        with pytest.raises(ValueError):
            lin.forward(x, out)
    with pytest.raises(ValueError, match="gradients=True"):
        lin.input_gradient(torch.zeros(4, 128, dtype=BF16, device=DEV))
    with pytest.raises(ValueError, match="accumulate needs out"):
        lin.weight_gradient(torch.zeros(4, 128, dtype=BF16, device=DEV), x, accumulate=True)
    with pytest.raises(ValueError):
        lin.weight_gradient(torch.zeros(3, 128, dtype=BF16, device=DEV), x)
    q, s, _ = C.weights(128, 256, seed=1)
    with pytest.raises(ValueError, match="weight_scale"):
        BlockLinear(q.to(DEV), s.t().contiguous().to(DEV))
    with pytest.raises(ValueError):
        BlockLinear(q, s)


def test_outputs_that_share_memory_with_inputs_are_refused():
    lin, w = layer(128, 128, seed=30, gradients=True)
    buf = torch.zeros(40, 300, dtype=BF16, device=DEV)
    x = C.activations(40, 128, seed=31)
    buf[:, :128] = x.to(DEV)
    for out in (buf[:, :128], buf[:, 127:255]):
        with pytest.raises(RuntimeError, match="shares memory"):
            lin.forward(buf[:, :128], out)
    lin.forward(buf[:, :128], buf[:, 128:256])  # other columns of the same rows
    C.assert_within(buf[:, 128:256], *C.product(C.quantised(x, 1), w))
    dw = torch.zeros(128, 128, device=DEV)
    with pytest.raises(RuntimeError, match="shares memory"):
        lin.weight_gradient(dw[:40], x.to(DEV), dw)


@pytest.mark.parametrize("T,N,K", [(1, 64, 64), (40, 256, 512), (65, 300, 200), (100, 1024, 2048), (333, 1024, 1024), (900, 700, 500),
                                   (2000, 256, 128)])
def test_backward_is_both_gradients(T, N, K):
    lin, _ = layer(N, K, seed=32, gradients=True)
    x, dy = C.activations(T, K, seed=33).to(DEV), C.activations(T, N, seed=34).to(DEV)
    dx, dw = lin.backward(dy, x)
    assert torch.equal(dx, lin.input_gradient(dy)) and torch.equal(dw, lin.weight_gradient(dy, x))
    acc = dw.clone()
    assert lin.backward(dy, x, acc, accumulate=True)[1] is acc and torch.equal(acc, dw + dw)
    with pytest.raises(ValueError, match="gradients=True"):
        layer(N, K, seed=32)[0].backward(dy, x)


@pytest.mark.parametrize("T,N,K", [(3, 40, 60), (40, 255, 130), (200, 129, 250), (2000, 256, 127)])
@pytest.mark.parametrize("dt,xt", [(F32, BF16), (BF16, F32)])
def test_backward_of_mixed_types(T, N, K, dt, xt):
    lin, w = layer(N, K, seed=35, gradients=True)
    x, dy = C.activations(T, K, seed=36, dtype=xt), C.activations(T, N, seed=37, dtype=dt)
    dx, dw = lin.backward(dy.to(DEV), x.to(DEV))
    C.assert_within(dx, *C.product(C.quantised(dy, 1), w.t().contiguous()), "dx")
    C.assert_within(dw, *C.outer(dy, x), "dw")


@pytest.mark.parametrize("T,N,K,dt", [(2000, 255, 130, BF16), (300, 129, 250, F32), (30, 40, 61, F32)])
def test_captured_backward_with_copies_and_splits(T, N, K, dt):
    lin, _ = layer(N, K, seed=38, gradients=True)
    x, dy = C.activations(T, K, seed=39, dtype=dt).to(DEV), C.activations(T, N, seed=40, dtype=dt).to(DEV)
    lin.backward(dy, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, dw = lin.backward(dy, x)
    for i in range(4):
        x.copy_(C.activations(T, K, seed=50 + i, dtype=dt))
        dy.copy_(C.activations(T, N, seed=60 + i, dtype=dt))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((dx, dw), lin.backward(dy, x)):
            assert torch.equal(a, b)
