"""Root-mean-square norm before a projection or the experts, with the residual's
addition and an output in 8 bits, and its gradients (include/netra_layers.h has the
formulas).

    n = rms_norm(x, weight, residual=stream, codes="rows")
    n.y                      # bf16 [T, H]: the router's input, or a projection's
    n.residual               # x + residual in the residual's type: the next block's residual
    n.codes, n.scale         # e4m3 [T, H] and fp32 [T, ceil(H/128)]: the bridges' input

codes="tiles" lays codes and scales out for BlockLinear.forward_codes. out= and
residual_out= may be x and residual themselves.

    dx, dw = rms_norm_gradients(dy, n.residual, weight, residual_gradient=g)

dx is the gradient of x and of residual alike; the codes are taken as y itself.
Nothing is recorded by autograd.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .layers import TYPES, check_rows, entry, launch, workspace

MAX_COLS = 16384
LAYOUTS = {"rows": 1, "tiles": 2}  # NETRA_CODES_ROWS, NETRA_CODES_TILES


class Norm(NamedTuple):
    y: torch.Tensor | None        # [T, H]
    residual: torch.Tensor        # what was normalised: x, or x + residual
    codes: torch.Tensor | None    # e4m3 [T, H], or tiles (uint8)
    scale: torch.Tensor | None    # fp32 [T, ceil(H/128)], or of the tiles


def _check_weight(weight: torch.Tensor, cols: int, device: torch.device) -> int:
    if weight.shape != (cols,) or weight.dtype not in TYPES or weight.device != device or not weight.is_contiguous():
        raise ValueError(f"weight: need contiguous torch.bfloat16 or torch.float32 ({cols},) on {device}, got "
                         f"{weight.dtype} {tuple(weight.shape)} on {weight.device}")
    return TYPES[weight.dtype]


def _check_input(name: str, x: torch.Tensor) -> None:
    if x.dim() != 2 or not x.is_cuda or not 1 <= x.shape[1] <= MAX_COLS:
        raise ValueError(f"{name}: need a bf16 or fp32 [T, H] GPU tensor with H in 1 .. {MAX_COLS}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6,
             offset: float = 0.0, out_type: torch.dtype | None = torch.bfloat16, codes: str | None = None,
             out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None) -> Norm:
    """x [T, H] (bf16 or fp32), residual likewise; weight [H] (bf16 or fp32), to which
    `offset` is added (1.0 for weights kept about zero). out_type: of y; None for no y."""
    _check_input("x", x)
    shape, device, x_type = x.shape, x.device, x.dtype
    rows, cols = shape
    x_stride = check_rows("x", x, shape, device)
    kind = _check_weight(weight, cols, device)
    # (empty_like is the quickest way to a tensor of one's shape: rows in order, however far apart x's are)
    if residual is not None:
        r_stride = check_rows("residual", residual, shape, device)
        if residual_out is None:
            residual_out, s_stride = torch.empty_like(residual), cols
        else:
            s_stride = check_rows("residual_out", residual_out, shape, device, (residual.dtype,))
        r_at, r_type, s_at = residual.data_ptr(), TYPES[residual.dtype], residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    else:
        r_at = r_type = r_stride = s_at = s_stride = 0
    if out is not None:
        y_stride = check_rows("out", out, shape, device)
        y_at, y_type = out.data_ptr(), TYPES[out.dtype]
    elif out_type is None:
        y_at = y_type = y_stride = 0
    elif out_type in TYPES:
        out = torch.empty_like(x, dtype=out_type)
        y_at, y_type, y_stride = out.data_ptr(), TYPES[out_type], cols
    else:
        raise ValueError(f"out_type: need torch.bfloat16, torch.float32 or None, got {out_type}")
    if codes is None:
        q = s = None
        q_at = s_scale = layout = 0
    else:
        layout = LAYOUTS.get(codes, 0)
        if layout == 1:
            q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
            s = x.new_empty((rows, -(-cols // 128)), dtype=torch.float32)
        elif layout == 2:
            q = x.new_empty(entry("netra_norm_code_bytes")(rows, cols, 2), dtype=torch.uint8)
            s = x.new_empty((-(-cols // 128), -(-rows // 16) * 16), dtype=torch.float32)
        else:
            raise ValueError(f"codes: need None, {' or '.join(map(repr, LAYOUTS))}, got {codes!r}")
        q_at, s_scale = q.data_ptr(), s.data_ptr()
    launch(entry("netra_norm_forward"), "netra_norm_forward", device, x.data_ptr(), TYPES[x_type], x_stride, r_at, r_type,
           r_stride, weight.data_ptr(), kind, offset, eps, s_at, s_stride, y_at, y_type, y_stride, q_at, s_scale, layout,
           rows, cols)
    return Norm(out, x if residual is None else residual_out, q, s)


def rms_norm_gradients(dy: torch.Tensor, r: torch.Tensor, weight: torch.Tensor, *,
                       residual_gradient: torch.Tensor | None = None, eps: float = 1e-6, offset: float = 0.0,
                       out: torch.Tensor | None = None, dw: torch.Tensor | None = None,
                       accumulate: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dw) of rms_norm: dy [T, H] the gradient of y, r what was normalised (Norm.residual),
    residual_gradient what flows into it besides. dx is of r's type (out= may be any of the
    inputs of that type), dw fp32 [H]; accumulate adds it to dw."""
    _check_input("r", r)
    shape, device, r_type = r.shape, r.device, r.dtype
    rows, cols = shape
    r_stride = check_rows("r", r, shape, device)
    dy_stride = check_rows("dy", dy, shape, device)
    kind = _check_weight(weight, cols, device)
    f_at = f_stride = 0
    if residual_gradient is not None:
        f_stride = check_rows("residual_gradient", residual_gradient, shape, device, (r_type,))
        f_at = residual_gradient.data_ptr()
    if out is None:
        out, o_stride = torch.empty_like(r), cols
    else:
        o_stride = check_rows("out", out, shape, device, (r_type,))
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs dw")
        dw = torch.empty_like(weight, dtype=torch.float32)
    elif dw.shape != (cols,) or dw.dtype != torch.float32 or dw.device != device or not dw.is_contiguous():
        raise ValueError(f"dw: need contiguous torch.float32 ({cols},) on {device}")
    need = entry("netra_norm_gradients_workspace")(rows, cols)
    ws, ws_ptr = workspace(need, device)
    launch(entry("netra_norm_gradients"), "netra_norm_gradients", device, dy.data_ptr(), TYPES[dy.dtype], dy_stride,
           r.data_ptr(), TYPES[r_type], r_stride, f_at, f_stride, weight.data_ptr(), kind, offset, eps, out.data_ptr(),
           o_stride, dw.data_ptr(), int(accumulate), rows, cols, ws_ptr, need)
    return out, dw
