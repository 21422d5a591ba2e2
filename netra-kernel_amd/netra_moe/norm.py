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


def _check_input(name: str, x: torch.Tensor) -> tuple[int, int]:
    if x.dim() != 2 or not x.is_cuda or not 1 <= x.shape[1] <= MAX_COLS:
        raise ValueError(f"{name}: need a bf16 or fp32 [T, H] GPU tensor with H in 1 .. {MAX_COLS}")
    return tuple(x.shape)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6,
             offset: float = 0.0, out_type: torch.dtype | None = torch.bfloat16, codes: str | None = None,
             out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None) -> Norm:
    """x [T, H] (bf16 or fp32), residual likewise; weight [H] (bf16 or fp32), to which
    `offset` is added (1.0 for weights kept about zero). out_type: of y; None for no y."""
    shape = rows, cols = _check_input("x", x)
    device = x.device
    x_stride = check_rows("x", x, shape, device)
    kind = _check_weight(weight, cols, device)
    if residual is not None:
        r_stride = check_rows("residual", residual, shape, device)
        if residual_out is None:
            residual_out, s_stride = residual.new_empty(shape), cols
        else:
            s_stride = check_rows("residual_out", residual_out, shape, device, (residual.dtype,))
        r_args = (residual.data_ptr(), TYPES[residual.dtype], r_stride)
        s_args = (residual_out.data_ptr(), s_stride)
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    else:
        r_args, s_args = (0, 0, 0), (0, 0)
    if out is not None:
        y, y_args = out, (out.data_ptr(), TYPES.get(out.dtype, 0), check_rows("out", out, shape, device))
    elif out_type is None:
        y, y_args = None, (0, 0, 0)
    elif out_type in TYPES:
        y = torch.empty(shape, dtype=out_type, device=device)
        y_args = (y.data_ptr(), TYPES[out_type], cols)
    else:
        raise ValueError(f"out_type: need torch.bfloat16, torch.float32 or None, got {out_type}")
    if codes is None:
        q = s = None
        q_args = (0, 0, 0)
    elif codes == "rows":
        q = torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)
        s = torch.empty((rows, -(-cols // 128)), dtype=torch.float32, device=device)
        q_args = (q.data_ptr(), s.data_ptr(), 1)
    elif codes == "tiles":
        q = torch.empty(entry("netra_norm_code_bytes")(rows, cols, 2), dtype=torch.uint8, device=device)
        s = torch.empty((-(-cols // 128), -(-rows // 16) * 16), dtype=torch.float32, device=device)
        q_args = (q.data_ptr(), s.data_ptr(), 2)
    else:
        raise ValueError(f"codes: need None, {' or '.join(map(repr, LAYOUTS))}, got {codes!r}")
    launch(entry("netra_norm_forward"), "netra_norm_forward", device, x.data_ptr(), TYPES[x.dtype], x_stride, *r_args,
           weight.data_ptr(), kind, offset, eps, *s_args, *y_args, *q_args, rows, cols)
    return Norm(y, x if residual is None else residual_out, q, s)


def rms_norm_gradients(dy: torch.Tensor, r: torch.Tensor, weight: torch.Tensor, *,
                       residual_gradient: torch.Tensor | None = None, eps: float = 1e-6, offset: float = 0.0,
                       out: torch.Tensor | None = None, dw: torch.Tensor | None = None,
                       accumulate: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dw) of rms_norm: dy [T, H] the gradient of y, r what was normalised (Norm.residual),
    residual_gradient what flows into it besides. dx is of r's type (out= may be any of the
    inputs of that type), dw fp32 [H]; accumulate adds it to dw."""
    shape = rows, cols = _check_input("r", r)
    device = r.device
    r_stride = check_rows("r", r, shape, device)
    dy_stride = check_rows("dy", dy, shape, device)
    kind = _check_weight(weight, cols, device)
    f_args = (0, 0)
    if residual_gradient is not None:
        f_args = (residual_gradient.data_ptr(), check_rows("residual_gradient", residual_gradient, shape, device, (r.dtype,)))
    if out is None:
        out, o_stride = r.new_empty(shape), cols
    else:
        o_stride = check_rows("out", out, shape, device, (r.dtype,))
    if dw is None:
        if accumulate:
            raise ValueError("accumulate needs dw")
        dw = torch.empty(cols, dtype=torch.float32, device=device)
    elif dw.shape != (cols,) or dw.dtype != torch.float32 or dw.device != device or not dw.is_contiguous():
        raise ValueError(f"dw: need contiguous torch.float32 ({cols},) on {device}")
    need = entry("netra_norm_gradients_workspace")(rows, cols)
    ws, ws_ptr = workspace(need, device)
    launch(entry("netra_norm_gradients"), "netra_norm_gradients", device, dy.data_ptr(), TYPES[dy.dtype], dy_stride,
           r.data_ptr(), TYPES[r.dtype], r_stride, *f_args, weight.data_ptr(), kind, offset, eps, out.data_ptr(), o_stride,
           dw.data_ptr(), int(accumulate), rows, cols, ws_ptr, need)
    return out, dw
