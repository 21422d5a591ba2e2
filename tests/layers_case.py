"""64-bit forms of the operators next to the MoE layer and the error bounds of
their fp32 computation, shared by the tests of netra_moe.linear and
netra_moe.balance.

Bounds. u = 2^-24 is the largest relative error of one fp32 rounding.

FP8 products: the matrix core aligns the products of 8 neighbouring k to the
largest exponent sum among them and drops what is below 2^-13 of it, so a group
of 8 is off by at most 8 * 2^-13 times its largest product, which is at most the
product of the two largest factors. Its fp32 sums (16 groups, then s_x * s_w and
an fma, then the blocks and the splits of the contraction) are off by at most
(18 + blocks + splits) u of the sum of the terms' magnitudes. Whole numbers small
enough to lose nothing are therefore exact.

The weight gradient's products of bf16 values are exact in fp32; its sum over the
tokens takes at most one rounding a token and split.

A bf16 output adds half a step, 2^-8 of the value."""
import numpy as np
import torch

U = 2.0 ** -24
INV_MAX = float(np.array([0x3B124925], dtype=np.uint32).view(np.float32)[0])
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
SPLITS = 64  # more than any variant uses


def blocks(n):
    return -(-n // 128)


def quantised(v, dim):
    """fp32 values v after the 1x128 rule along `dim`, as float64 (NaN where the
    128-group holds an infinity or NaN)."""
    v = v.detach().to("cpu", torch.float32).movedim(dim, -1)
    n = v.shape[-1]
    p = torch.nn.functional.pad(v, (0, -n % 128)).unflatten(-1, (-1, 128))
    amax = p.abs().amax(-1, keepdim=True)
    scale = torch.where(torch.isfinite(amax), amax.clamp_min(1e-10) * torch.tensor(INV_MAX), torch.nan)
    q = (p * (1.0 / scale)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (q.double() * scale.double()).flatten(-2)[..., :n].movedim(-1, dim)


def weights(n, k, seed, std=0.02):
    """e4m3 codes [n, k] and scales (host), and the values they stand for (float64)."""
    g = torch.Generator().manual_seed(seed)
    w = torch.zeros(blocks(n) * 128, blocks(k) * 128)
    w[:n, :k] = torch.randn(n, k, generator=g) * std
    b = w.view(blocks(n), 128, blocks(k), 128)
    scale = b.abs().amax((1, 3), keepdim=True).clamp_min(1e-10) * torch.tensor(INV_MAX)
    q = (b * (1.0 / scale)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    deq = (q.double() * scale.double()).view_as(w)[:n, :k]
    return q.view(w.shape)[:n, :k].contiguous(), scale.view(blocks(n), blocks(k)), deq


def activations(t, k, seed, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g) * std
    x[:, 3::37] *= 25.0
    return x.to(dtype)


def group_max(v):
    return torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 8)).unflatten(1, (-1, 8)).amax(2)


def product(a, b):
    """a b^T in float64 for quantised a, b, and the bound of the FP8 product by 128-blocks."""
    exact = a @ b.t()
    fp32 = (18 + blocks(a.shape[1]) + SPLITS) * U * (a.abs() @ b.abs().t())
    return exact, 8 * 2.0 ** -13 * (group_max(a) @ group_max(b).t()) + fp32


def outer(dy, x):
    """dy^T x in float64 of the bf16 values, and the bound of its fp32 sum."""
    dy, x = (v.detach().cpu().to(torch.bfloat16).double() for v in (dy, x))
    magnitude = torch.nan_to_num(dy.abs(), posinf=0).t() @ torch.nan_to_num(x.abs(), posinf=0)
    return dy.t() @ x, (dy.shape[0] + SPLITS) * U * magnitude


def assert_within(got, want, bound, what=""):
    """Every element within the bound and half a step of its type; NaN where NaN."""
    half = HALF_STEP[got.dtype]
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    limit = bound + half * (want.abs() + bound)
    off = torch.where(torch.isnan(want) | (got == want), 0.0, (got - want).abs() - limit)
    worst = int(off.argmax()) if off.numel() else 0
    assert not off.numel() or off.max() <= 0, \
        f"{what}: {got.reshape(-1)[worst]} for {want.reshape(-1)[worst]}, bound {limit.reshape(-1)[worst]}"


def counts(ids, experts, mask=None):
    ids = ids.cpu().numpy()
    if mask is not None:
        ids = ids[mask.cpu().numpy().astype(bool)]
    flat = ids.reshape(-1)
    return np.bincount(flat[(flat >= 0) & (flat < experts)], minlength=experts)


def balance(logits, counts_, bias=None, mask=None, coefficient=1.0):
    """(loss, gradient) in float64; rows that are all -inf add nothing."""
    z = logits.detach().cpu().double()
    T, E = z.shape
    live = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu().bool()
    z = torch.where(live[:, None], z, 0.0)
    if bias is not None:  # the sum is held in fp32, like the router's own
        z = (z.float() + bias.cpu()).double()
    c = torch.as_tensor(np.asarray(counts_), dtype=torch.float64)
    f = c * (E / c.sum()) if c.sum() else c * 0
    empty = (z == -torch.inf).all(1)
    p = torch.softmax(torch.where(empty[:, None], 0.0, z), 1)
    p = torch.where((live & ~empty)[:, None], p, 0.0)
    s = (p * f).sum(1, keepdim=True)
    scale = coefficient / int(live.sum()) if live.any() else 0.0
    return float(s.sum() * scale), p * (f - s) * scale, p, f, s, scale
