"""Low-rank adapters of many requests beside a shared projection (include/netra_layers.h has the
formulas).

    adapters = LowRankAdapters(a, b, scale)      # a [L, r, K], b [L, N, r], scale fp32 [L]
    plan = adapters.plan(ids)                    # int32 [T]: each token's adapter, anything else for none
    y = proj.forward(x, adapters=adapters, plan=plan)    # BlockLinear, with its adapters
    adapters.add(y, x, plan)                     # or beside a projection of one's own: y + s B (A x)

The plan sorts a batch's tokens by adapter. It depends on the ids, the number of tokens and the number of
adapters alone: a serving step makes one and uses it for all its projections. Making it launches one kernel
and waits for nothing, so it may be captured into a graph with the calls that use it. A serving operator: there is
no backward pass.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from .layers import TYPES, check_rows, entry, launch, workspace

MAX_ADAPTERS = 1024
MAX_RANK = 128


class AdapterPlan(NamedTuple):
    data: torch.Tensor
    tokens: int
    adapters: int


def make_plan(ids: torch.Tensor, adapters: int) -> AdapterPlan:
    """The plan of a batch for any set of so many adapters."""
    if ids.dim() != 1 or ids.dtype != torch.int32 or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("ids: need a contiguous int32 [T] GPU tensor")
    if not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"adapters: need 1 .. {MAX_ADAPTERS}, got {adapters}")
    tokens = ids.shape[0]
    need = entry("netra_adapters_plan_bytes")(tokens, adapters)
    data = torch.empty(need, dtype=torch.uint8, device=ids.device)
    launch(entry("netra_adapters_plan"), "netra_adapters_plan", ids.device, ids.data_ptr(), tokens, adapters,
           data.data_ptr(), need)
    return AdapterPlan(data, tokens, adapters)


class LowRankAdapters:
    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None = None):
        """a [L, r, K] and b [L, N, r], both bf16 or both fp32 (rounded to bf16), on the GPU; scale fp32
        [L] (default: ones). All are copied into the object."""
        if a.dim() != 3 or b.dim() != 3 or a.dtype not in TYPES or b.dtype != a.dtype or not a.is_cuda \
                or b.device != a.device or not a.is_contiguous() or not b.is_contiguous() or a.numel() == 0 or b.numel() == 0:
            raise ValueError("LowRankAdapters needs contiguous a [L, r, K] and b [L, N, r] of one type (bf16 or fp32) on one GPU")
        self.count, self.rank, self.K = a.shape
        self.N = b.shape[1]
        if b.shape != (self.count, self.N, self.rank):
            raise ValueError(f"b: need [{self.count}, N, {self.rank}] beside a {tuple(a.shape)}, got {tuple(b.shape)}")
        if not self.count <= MAX_ADAPTERS or not self.rank <= MAX_RANK:
            raise ValueError(f"need at most {MAX_ADAPTERS} adapters of rank {MAX_RANK}, got {self.count} of {self.rank}")
        self.device = a.device
        if scale is None:
            scale = torch.ones(self.count, dtype=torch.float32, device=self.device)
        if scale.shape != (self.count,) or scale.dtype != torch.float32 or scale.device != self.device:
            raise ValueError(f"scale: need torch.float32 ({self.count},) on {self.device}")
        self.scale = scale.contiguous().clone()
        size = entry("netra_adapters_packed_bytes")
        sizes = (self.count, self.rank, self.N, self.K)
        self.a, self.b = (torch.empty(size(*sizes, which), dtype=torch.uint8, device=self.device) for which in (0, 1))
        launch(entry("netra_adapters_pack"), "netra_adapters_pack", self.device, a.data_ptr(), b.data_ptr(), TYPES[a.dtype],
               self.a.data_ptr(), self.b.data_ptr(), *sizes)
        self._add, self._need = entry("netra_adapters_add"), entry("netra_adapters_add_workspace")
        self._weights = (self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr())

    @classmethod
    def from_pairs(cls, pairs: Sequence[tuple[torch.Tensor, torch.Tensor]], scale: torch.Tensor | None = None) -> "LowRankAdapters":
        """Adapters (a [r, K], b [N, r]) of different ranks, filled with zeros to the largest (with which a row of x that
        holds an infinity or NaN gives NaN)."""
        if not pairs:
            raise ValueError("from_pairs needs an adapter")
        for i, (a, b) in enumerate(pairs):
            if a.dim() != 2 or b.dim() != 2 or b.shape[1] != a.shape[0]:
                raise ValueError(f"pairs[{i}]: need a [r, K] and b [N, r], got {tuple(a.shape)} and {tuple(b.shape)}")
        rank = max(a.shape[0] for a, _ in pairs)
        fill = torch.nn.functional.pad
        return cls(torch.stack([fill(a, (0, 0, 0, rank - a.shape[0])) for a, _ in pairs]),
                   torch.stack([fill(b, (0, rank - b.shape[1])) for _, b in pairs]), scale)

    def plan(self, ids: torch.Tensor) -> AdapterPlan:
        return make_plan(ids, self.count)

    def add(self, y: torch.Tensor, x: torch.Tensor, plan: AdapterPlan, out: torch.Tensor | None = None) -> torch.Tensor:
        """y bf16 [T, N] + the adapters of x bf16 or fp32 (rounded to bf16) [T, K], bf16 [T, N]; out may be y."""
        data, tokens, adapters = plan
        if adapters != self.count or data.device != self.device:
            raise ValueError(f"plan: need one of {self.count} adapters on {self.device}, got {adapters} on {data.device}")
        x_stride = check_rows("x", x, (tokens, self.K), self.device)
        y_stride = check_rows("y", y, (tokens, self.N), self.device, (torch.bfloat16,))
        if out is None:
            out, out_stride = torch.empty_like(y), self.N
        else:
            out_stride = check_rows("out", out, (tokens, self.N), self.device, (torch.bfloat16,))
        need = self._need(tokens, adapters, self.rank, self.N, self.K)
        ws, ws_ptr = workspace(need, self.device)
        launch(self._add, "netra_adapters_add", self.device, x.data_ptr(), TYPES[x.dtype], x_stride, *self._weights,
               data.data_ptr(), y.data_ptr(), y_stride, out.data_ptr(), out_stride, tokens, adapters, self.rank, self.N,
               self.K, ws_ptr, need)
        return out
