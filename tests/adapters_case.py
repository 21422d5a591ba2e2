"""64-bit form of netra_moe.adapters and the bound of its fp32 computation (u = 2^-24).

A x is a sum of k products of bf16 values, exact in fp32 each: k additions in the matrix core and over
waves and splits, (k + 40) u of the sum of magnitudes. It is scaled (u) and split into two bf16 values, off by
2^-16 of it at most (2^-8 of what the first left, itself at most 2^-8). The sum over the rank adds 2 (2 rank + 8) u of
its magnitudes, as each value comes in two parts."""
import torch

from layers_case import U, assert_within  # noqa: F401


def adapters(L, r, k, n, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(L, r, k, generator=g) / k ** 0.5).to(dtype), (torch.randn(L, n, r, generator=g) / r ** 0.5).to(dtype),
            torch.rand(L, generator=g) + 0.5)


def add(y, x, a, b, scale, ids):
    """(out in float64, bound before its rounding)."""
    bf = lambda v: v.detach().cpu().to(torch.bfloat16).double()  # noqa: E731
    x, y, a, b, scale, ids = bf(x), bf(y), bf(a), bf(b), scale.cpu().double(), ids.cpu().long()
    out, bound = y.clone(), torch.zeros_like(y)
    k, r = a.shape[2], a.shape[1]
    for l in range(len(a)):
        t = (ids == l).nonzero().view(-1)
        if not len(t):
            continue
        u, size = x[t] @ a[l].t() * scale[l], x[t].abs() @ a[l].abs().t() * scale[l].abs()
        out[t] += u @ b[l].t()
        off = (k + 41) * U * size + 2.0 ** -16 * u.abs()
        bound[t] = off @ b[l].abs().t() + (4 * r + 16) * U * (u.abs() @ b[l].abs().t()) + 2 * U * (y[t].abs() + out[t].abs())
    return out, bound
