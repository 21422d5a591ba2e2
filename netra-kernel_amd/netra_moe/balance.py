"""Per-expert route counts and the router's balance loss with its gradient
(include/netra_layers.h has the formulas).

The router's logits and top-k ids come from MoELayer (expose=("logits",
"topk_ids")) or from a caller's own router: the layer's logits have the
shared expert's gate as their last column (pass logits[:, :E]) and its ids the
shared expert as id E in the last slot, which is not counted.

    counts = expert_counts(topk_ids, E)
    r = balance_loss(logits, topk_ids, coefficient=0.01)
    r.loss, r.counts, r.grad            # grad: with respect to logits, in their type

Nothing is recorded by autograd: r.grad goes to logits.backward(r.grad) of a caller
whose router torch differentiates.

Over several ranks the loss uses the whole job's counts: sum expert_counts()
over the ranks and pass the result as counts=.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .layers import TYPES, check_rows, entry, launch, workspace

MAX_EXPERTS = 1024


class BalanceLoss(NamedTuple):
    loss: torch.Tensor            # fp32, one element
    counts: torch.Tensor          # int32 [E]
    grad: torch.Tensor | None     # as logits, or None


def _check_mask(mask: torch.Tensor | None, tokens: int, device: torch.device) -> int:
    if mask is None:
        return 0
    if tuple(mask.shape) != (tokens,) or mask.dtype not in (torch.bool, torch.uint8) or mask.device != device \
            or not mask.is_contiguous():
        raise ValueError(f"mask: need contiguous torch.bool or torch.uint8 ({tokens},) on {device}, got {mask.dtype} "
                         f"{tuple(mask.shape)} on {mask.device}")
    return mask.data_ptr()


def _check_counts(name: str, counts: torch.Tensor, experts: int, device: torch.device) -> None:
    if tuple(counts.shape) != (experts,) or counts.dtype != torch.int32 or counts.device != device \
            or not counts.is_contiguous():
        raise ValueError(f"{name}: need contiguous torch.int32 ({experts},) on {device}, got {counts.dtype} "
                         f"{tuple(counts.shape)} on {counts.device}")


def _check_ids(ids: torch.Tensor, tokens: int | None, device: torch.device) -> int:
    if not ids.is_cuda or ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError("topk_ids: need an int32 [T, slots] GPU tensor")
    return check_rows("topk_ids", ids, (ids.shape[0] if tokens is None else tokens, ids.shape[1]), device, (torch.int32,))


def _check_experts(experts: int) -> None:
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts: need 1 .. {MAX_EXPERTS}, got {experts}")


def expert_counts(topk_ids: torch.Tensor, experts: int, *, mask: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """Routes per expert, int32 [experts], of ids int32 [T, slots]; ids outside
    0 .. experts - 1 and tokens whose mask is false are not counted. accumulate
    adds to out (the load over several calls)."""
    _check_experts(experts)
    stride = _check_ids(topk_ids, None, topk_ids.device)
    device, (tokens, slots) = topk_ids.device, topk_ids.shape
    m = _check_mask(mask, tokens, device)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = topk_ids.new_empty(experts)
    else:
        _check_counts("out", out, experts, device)
    need = entry("netra_router_counts_workspace")(tokens, slots, experts)
    ws, ws_ptr = workspace(need, device)
    launch(entry("netra_router_counts"), "netra_router_counts", device, topk_ids.data_ptr(), stride, m, tokens, slots,
           experts, out.data_ptr(), int(accumulate), ws_ptr, need)
    return out


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor | None = None, *, counts: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, coefficient: float = 1.0,
                 grad: bool = True) -> BalanceLoss:
    """Balance loss of logits bf16 or fp32 [T, E] and its gradient. Give topk_ids
    (counted here) or counts (int32 [E], for instance summed over ranks). bias:
    fp32 [E] added to the logits before the softmax, as the layer's router does;
    a constant. mask: tokens that count."""
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits: need a bf16 or fp32 [T, E] GPU tensor")
    device, (tokens, experts) = logits.device, logits.shape
    _check_experts(experts)
    logits_stride = check_rows("logits", logits, (tokens, experts), device)
    if (topk_ids is None) == (counts is None):
        raise ValueError("balance_loss needs either topk_ids or counts")
    m = _check_mask(mask, tokens, device)
    if bias is not None and (tuple(bias.shape) != (experts,) or bias.dtype != torch.float32 or bias.device != device
                             or not bias.is_contiguous()):
        raise ValueError(f"bias: need contiguous torch.float32 ({experts},) on {device}")
    if topk_ids is not None:
        stride = _check_ids(topk_ids, tokens, device)
        slots, ids = topk_ids.shape[1], topk_ids.data_ptr()
        counts = topk_ids.new_empty(experts)
    else:
        _check_counts("counts", counts, experts, device)
        slots, ids, stride = 0, 0, 0
    loss = torch.empty((), dtype=torch.float32, device=device)
    g = logits.new_empty((tokens, experts)) if grad else None
    need = entry("netra_router_balance_workspace")(tokens, slots, experts)
    ws, ws_ptr = workspace(need, device)
    launch(entry("netra_router_balance"), "netra_router_balance", device, logits.data_ptr(), TYPES[logits.dtype],
           logits_stride, bias.data_ptr() if bias is not None else 0, ids, stride, slots, m, tokens, experts,
           coefficient, counts.data_ptr(), loss.data_ptr(), g.data_ptr() if grad else 0, experts, ws_ptr, need)
    return BalanceLoss(loss, counts, g)
