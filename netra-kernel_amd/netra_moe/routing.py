"""Routing to experts and its gradient (include/netra_layers.h has the formulas).

    r = route(logits, 8)                                    # softmax, the 8 best, weights renormalised
    r = route(logits, 8, scoring="sigmoid", selection_bias=bias, groups=8, top_groups=4,
              group_score="top2", scale=2.5)
    r = route(layer_logits, 8, shared=True)                 # logits [T, E + 1] as MoELayer's: the shared expert
                                                            # as id E with its sigmoid gate in the last slot
    r.ids, r.weights                                        # int32 and fp32 [T, 8 (+ 1)]

ids feed expert_counts, balance_loss and the bridges. selection_bias moves the choice and not
the weights (MoELayer's router_bias is added to the logits instead: give logits + bias for that). A bias of -inf takes an
expert out at no cost; a large finite one (-1e9) does so too and makes the call several times as long.

    g = route_gradient(dweights, logits, r.ids)             # of the logits' type and shape
    route_gradient(dweights, logits, r.ids, out=b.grad, accumulate=True)   # adds to the balance loss's

Nothing is recorded by autograd. selection_bias and the choice itself have no gradient.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .balance import MAX_EXPERTS, _check_mask
from .layers import TYPES, check_rows, entry, launch

MAX_SLOTS = 16
SCORING = {"softmax": 0, "sigmoid": 1}   # NETRA_SOFTMAX, NETRA_SIGMOID
GROUP_SCORE = {"max": 0, "top2": 1}      # NETRA_GROUP_MAX, NETRA_GROUP_TOP2


class Routing(NamedTuple):
    ids: torch.Tensor      # int32 [T, k + shared]
    weights: torch.Tensor  # fp32 [T, k + shared]


def _check_logits(logits: torch.Tensor, shared: bool) -> tuple[int, int]:
    if logits.dim() != 2 or not logits.is_cuda or not 1 <= logits.shape[1] - shared <= MAX_EXPERTS:
        raise ValueError(f"logits: need a bf16 or fp32 [T, E{' + 1' if shared else ''}] GPU tensor with E in 1 .. {MAX_EXPERTS}")
    return logits.shape[0], logits.shape[1] - shared


def _number(name: str, value: str, known: dict[str, int]) -> int:
    if value not in known:
        raise ValueError(f"{name}: need {' or '.join(map(repr, known))}, got {value!r}")
    return known[value]


def route(logits: torch.Tensor, k: int, *, scoring: str = "softmax", selection_bias: torch.Tensor | None = None,
          groups: int = 1, top_groups: int | None = None, group_score: str = "max", renormalise: bool = True,
          scale: float = 1.0, shared: bool = False, mask: torch.Tensor | None = None) -> Routing:
    """logits bf16 or fp32 [T, E] ([T, E + 1] with shared). top_groups: of `groups`, how many are
    kept (default: all). mask: tokens that are routed; the others get ids -1 and weights 0."""
    tokens, experts = _check_logits(logits, shared)
    device = logits.device
    stride = check_rows("logits", logits, (tokens, experts + shared), device)
    m = _check_mask(mask, tokens, device)
    slots = k + shared
    if not 1 <= k <= min(experts, MAX_SLOTS - shared):
        raise ValueError(f"k: need 1 .. {min(experts, MAX_SLOTS - shared)}, got {k}")
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= groups <= MAX_SLOTS or experts % groups or not 1 <= top_groups <= groups \
            or k > top_groups * (experts // groups):
        raise ValueError(f"groups, top_groups: need 1 .. {MAX_SLOTS} groups that divide {experts} experts and {k} experts "
                         f"or more in the top groups, got {groups} and {top_groups}")
    bias = 0
    if selection_bias is not None:
        if selection_bias.shape != (experts,) or selection_bias.dtype != torch.float32 or selection_bias.device != device \
                or not selection_bias.is_contiguous():
            raise ValueError(f"selection_bias: need contiguous torch.float32 ({experts},) on {device}")
        bias = selection_bias.data_ptr()
    ids = logits.new_empty((tokens, slots), dtype=torch.int32)
    weights = torch.empty_like(ids, dtype=torch.float32)
    launch(entry("netra_router_select"), "netra_router_select", device, logits.data_ptr(), TYPES[logits.dtype], stride, bias,
           m, tokens, experts, k, int(shared), _number("scoring", scoring, SCORING), groups, top_groups,
           _number("group_score", group_score, GROUP_SCORE), int(renormalise), scale, ids.data_ptr(), slots,
           weights.data_ptr(), slots)
    return Routing(ids, weights)


def route_gradient(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *, scoring: str = "softmax",
                   renormalise: bool = True, scale: float = 1.0, shared: bool = False,
                   mask: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   accumulate: bool = False) -> torch.Tensor:
    """The gradient with respect to logits of route()'s weights for its ids, given theirs: dweights
    fp32 [T, k + shared]. The other arguments are route()'s. accumulate adds to out."""
    tokens, experts = _check_logits(logits, shared)
    device = logits.device
    stride = check_rows("logits", logits, (tokens, experts + shared), device)
    m = _check_mask(mask, tokens, device)
    slots = dweights.shape[1] if dweights.dim() == 2 else 0
    k = slots - shared
    if not 1 <= k <= min(experts, MAX_SLOTS - shared):
        raise ValueError(f"dweights: need fp32 [T, k{' + 1' if shared else ''}] with k in 1 .. {min(experts, MAX_SLOTS - shared)}")
    d_stride = check_rows("dweights", dweights, (tokens, slots), device, (torch.float32,))
    i_stride = check_rows("ids", ids, (tokens, slots), device, (torch.int32,))
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out, o_stride = torch.empty_like(logits), experts + shared
    else:
        o_stride = check_rows("out", out, (tokens, experts + shared), device, (logits.dtype,))
    launch(entry("netra_router_select_gradient"), "netra_router_select_gradient", device, dweights.data_ptr(), d_stride,
           logits.data_ptr(), TYPES[logits.dtype], stride, ids.data_ptr(), i_stride, m, tokens, experts, k, int(shared),
           _number("scoring", scoring, SCORING), int(renormalise), scale, out.data_ptr(), o_stride, int(accumulate))
    return out
