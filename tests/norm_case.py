"""64-bit forms of netra_moe.norm and the bounds of its fp32 computation.

u = 2^-24. The sum of squares of a row is held by at most 1024 lanes of 16 values each: 16 sums in
a lane, 6 over the wave, 15 over the waves, so it is off by 38 u of itself; with the mean's and eps's
roundings and the root (which halves them) and quotient behind it rstd is off by less than 24 u, and y =
r * rstd * (w + offset) by 27 u of itself: 30 u below. The row's dot product is off by the same 38 u and
its products' 2 u, of the sum of its terms' magnitudes."""
import torch

from layers_case import HALF_STEP, U, INV_MAX, assert_within, blocks  # noqa: F401

Y = 30 * U
MOST = torch.float32


def normalised(x, residual):
    """r as the operator holds it (its rounding is part of the operator), in the residual's type."""
    x = x.cpu()
    return x if residual is None else (x.float() + residual.cpu().float()).to(residual.dtype)


def norm(r, w, eps=1e-6, offset=0.0):
    r, w = r.double(), w.cpu().float().double()
    return r / (r.square().mean(1, keepdim=True) + eps).sqrt() * (w + offset)


def check_y(got, want, what="y"):
    assert_within(got, want, Y * want.abs() + 1e-38, what)


def check_codes(codes, scale, want):
    """codes: the values of the e4m3 codes [T, H] (float64), scale [T, blocks], both on the host, against y."""
    T, H = want.shape
    p = torch.nn.functional.pad(want, (0, -H % 128)).view(T, blocks(H), 128)
    amax = p.abs().amax(2)
    bad = ~torch.isfinite(amax)
    assert torch.equal(torch.isnan(scale), bad)
    s64 = amax.clamp_min(1e-10) * INV_MAX
    off = (scale.double() - s64).abs() - (Y + 2 * U) * s64
    assert not (off[~bad] > 0).any()
    q = (p / s64[:, :, None]).view(T, -1)[:, :H]
    fine = ~bad.repeat_interleave(128, 1)[:, :H]
    # half a step of e4m3, 2^-4 of the value or 2^-10 among the smallest; the quotient is off by y's, the scale's and its own roundings
    limit = torch.maximum(q.abs() * 2.0 ** -4, torch.full_like(q, 2.0 ** -10)) + q.abs() * (2 * Y + 6 * U)
    worst = ((codes - q).abs() - limit)[fine]
    assert worst.numel() == 0 or worst.max() <= 0


def untile(codes, scale, rows, cols):
    """Values of tile16x128 codes and scales [blocks, rows up to 16] as (codes [rows, cols], scale [rows, blocks])."""
    kb = blocks(cols)
    v = codes.cpu().view(torch.float8_e4m3fn).double().view(-1, kb, 2, 4, 16, 16)  # row tile, block, half, quarter, row, column
    v = v.permute(0, 4, 1, 3, 2, 5).reshape(-1, kb * 128)
    return v[:rows, :cols], scale.cpu().t()[:rows]


def gradients(dy, r, w, flow, eps=1e-6, offset=0.0):
    """(dr, dw) in float64 and their bounds before rounding to a type."""
    dy, r, w = (v.detach().cpu().double() for v in (dy, r, w))
    w = w + offset
    rstd = 1.0 / (r.square().mean(1, keepdim=True) + eps).sqrt()
    xh, g = r * rstd, dy * w
    c = (g * xh).mean(1, keepdim=True)
    dr = rstd * (g - xh * c)
    dr_bound = rstd * (34 * U * g.abs() + xh.abs() * (100 * U * (g * xh).abs().mean(1, keepdim=True)))
    if flow is not None:
        flow = flow.cpu().double()
        dr = dr + flow
        dr_bound = dr_bound + 2 * U * (flow.abs() + dr.abs())
    return dr, (dy * xh).sum(0), dr_bound, (r.shape[0] + 60) * U * (dy * xh).abs().sum(0)
