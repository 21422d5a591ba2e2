"""64-bit forms of netra_moe.routing and the bounds of its fp32 computation (u = 2^-24).

The choice has no tolerance. A sigmoid is off by 7 u of itself (exp 4 u, sum and quotient 1 u each and a spare one). An
exponential of z - m is off by 4 u and, for the difference's rounding, |z - m| u. Sums of at most 1024 terms
by 64 lanes of 16 are off by 22 u, of 16 choices by 4 u. A weight is a quotient of two of these times the scale:
30 u, and 2 |z - m| u for a softmax; 40 u below. What is below 2^-126 may be 0."""
import torch

from layers_case import U, assert_within  # noqa: F401

TINY = 2.0 ** -126


def inputs(T, E, seed, dtype=torch.bfloat16, shared=False, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(T, E + shared, generator=g) * spread + torch.randn(E + shared, generator=g)
    return z.to(dtype)


def scores(z, scoring):
    """Of logits [T, E] in float64; rows that are all -inf have scores 0."""
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    empty = (z == -torch.inf).all(1, keepdim=True)
    return torch.where(empty, 0.0, torch.softmax(torch.where(empty, 0.0, z), 1))


def first_best(c, n):
    """Indexes of the n largest of each row, in order; ties to the lower index, NaN as -inf."""
    c = torch.where(torch.isnan(c), -torch.inf, c)
    return torch.sort(-c, dim=1, stable=True).indices[:, :n]


def choose(z, k, scoring="softmax", bias=None, groups=1, top_groups=1, group_score="max"):
    T, E = z.shape
    z = z.cpu().double()
    grouped = 1 < groups and top_groups < groups
    if bias is None and not (grouped and group_score == "top2"):
        c = z
    else:
        c = scores(z, scoring) + (0.0 if bias is None else bias.cpu().double())
    c = torch.where(torch.isnan(c), -torch.inf, c)
    away = torch.zeros((T, E), dtype=torch.bool)
    if grouped:
        parts = c.view(T, groups, E // groups).sort(2, descending=True).values
        value = parts[:, :, 0] + parts[:, :, 1] if group_score == "top2" else parts[:, :, 0]
        keep = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, first_best(value, top_groups), True)
        away = ~keep.repeat_interleave(E // groups, 1)
    # (what is away comes behind a -inf that is not)
    order = torch.sort(torch.where(away, -torch.inf, c), dim=1, descending=True, stable=True).indices
    behind = torch.sort(torch.gather(away, 1, order).long(), dim=1, stable=True).indices
    return torch.gather(order, 1, behind)[:, :k]


def weights(z, ids, scoring="softmax", renormalise=True, scale=1.0, shared=False):
    """(weights in float64, bound)."""
    z = z.cpu().double()
    E = z.shape[1] - shared
    x = z[:, :E]
    chosen = torch.gather(x, 1, ids)
    rel = torch.full_like(chosen, 40 * U)
    if renormalise and scoring == "softmax":
        s = scores(chosen, scoring)
        w = s * scale
    else:
        s = torch.gather(scores(x, scoring), 1, ids)
        total = s.sum(1, keepdim=True) if renormalise else 1.0
        w = torch.where(torch.as_tensor(total == 0.0), 0.0, s / total) * scale if renormalise else s * scale
    if scoring == "softmax":
        top = (chosen if renormalise else x).amax(1, keepdim=True)
        rel = rel + 2 * U * torch.nan_to_num((chosen - top).abs(), nan=0.0, posinf=0.0).amax(1, keepdim=True).clamp_max(200)
    if shared:
        w = torch.cat([w, torch.sigmoid(z[:, E:])], 1)
        rel = torch.cat([rel, torch.full((len(z), 1), 10 * U, dtype=torch.float64)], 1)
    return w, rel * w.abs() + 4 * max(1.0, abs(scale)) * TINY


def gradient(dw, z, ids, scoring="softmax", renormalise=True, scale=1.0, shared=False):
    """(gradient of the logits in float64, bound before rounding). The bound: 100 u, and for a
    softmax 4 |z - m| u, of the sums with every difference v_i - v_j replaced by |v_i| + |v_j|."""
    z, dw, ids = z.cpu().double(), dw.cpu().double(), ids.cpu().long()
    T, E = z.shape[0], z.shape[1] - shared
    k = dw.shape[1] - shared
    x, ids, v = z[:, :E], ids[:, :k], dw[:, :k] * scale
    there = (ids >= 0) & (ids < E)
    at = torch.where(there, ids, 0)
    v = torch.where(there, v, 0.0)
    chosen = torch.where(there, torch.gather(x, 1, at), -torch.inf)
    grad, bound = torch.zeros(T, E + shared, dtype=torch.float64), torch.zeros(T, E + shared, dtype=torch.float64)
    add = lambda g, b: (grad[:, :E].scatter_add_(1, at, torch.where(there, g, 0.0)),  # noqa: E731
                        bound[:, :E].scatter_add_(1, at, torch.where(there, b, 0.0)))
    rel = 100 * U
    if scoring == "sigmoid":
        s = torch.where(there, torch.sigmoid(chosen), 0.0)
        slope = s * torch.sigmoid(-chosen)
        slope = torch.where(there, slope, 0.0)
        if renormalise:
            total = s.sum(1, keepdim=True)
            inv = torch.where(total == 0.0, 0.0, 1.0 / total)
            d = (s[:, None, :] * (v[:, :, None] - v[:, None, :])).sum(2) * inv * inv
            m = (s[:, None, :] * (v.abs()[:, :, None] + v.abs()[:, None, :])).sum(2) * inv * inv
        else:
            d, m = v, v.abs()
        add(d * slope, rel * m * slope)
    elif renormalise:
        p = torch.where(there, scores(chosen, "softmax"), 0.0)
        far = torch.nan_to_num((chosen - chosen.amax(1, keepdim=True)).abs(), nan=0.0, posinf=0.0).amax(1, keepdim=True).clamp_max(200)
        d = (p[:, None, :] * (v[:, :, None] - v[:, None, :])).sum(2)
        m = (p[:, None, :] * (v.abs()[:, :, None] + v.abs()[:, None, :])).sum(2)
        add(p * d, (rel + 4 * U * far) * p * m)
    else:
        p = scores(x, "softmax")
        far = torch.nan_to_num((x - x.amax(1, keepdim=True)).abs(), nan=0.0, posinf=0.0).amax(1, keepdim=True).clamp_max(200)
        full = torch.zeros(T, E, dtype=torch.float64).scatter_add_(1, at, v)
        size = torch.zeros(T, E, dtype=torch.float64).scatter_add_(1, at, v.abs())
        grad[:, :E] = p * (full - (p * full).sum(1, keepdim=True))
        for i in range(k):  # of the chosen the differences, which keep their bits where one p is nearly 1
            e = at[:, i:i + 1]
            mine = torch.gather(full, 1, e)
            g = torch.gather(p, 1, e) * (p * (mine - full)).scatter(1, e, 0.0).sum(1, keepdim=True)
            grad[:, :E] = torch.where(there[:, i:i + 1], grad[:, :E].scatter(1, e, g), grad[:, :E])
        bound[:, :E] = (rel + 4 * U * far) * p * (size + (p * size).sum(1, keepdim=True))
    if shared:
        g = z[:, E:]
        grad[:, E:] = dw[:, k:] * torch.sigmoid(g) * torch.sigmoid(-g)
        bound[:, E:] = rel * grad[:, E:].abs()
    return grad, bound + 4 * TINY * max(1.0, abs(scale)) * dw.abs().amax().clamp_min(1.0)
