"""Block-FP8 linear layer: the dense projections of a block-FP8 checkpoint.

y = x W^T with W [N, K] in e4m3 and one fp32 scale per 128x128 block. x is
quantised inside the call by the MoE layer's 1x128 rule and the product runs on
the FP8 matrix cores with fp32 accumulation (include/netra_layers.h has the
formulas). N and K need not be multiples of 128.

    layer = BlockLinear(weight, weight_scale)              # codes as the checkpoint holds them
    layer = BlockLinear.from_checkpoint(tensors, "model.layers.3.self_attn.o_proj", device)
    y = layer.forward(x)

Training: BlockLinear(..., gradients=True) also keeps W^T, and

    dx, dw = layer.backward(dy, x)

gives the gradients with respect to the input (bf16; dy is quantised per 1x128)
and the weight (fp32; a bf16 product over the tokens, fp32 inputs rounded to bf16).
Nothing is recorded by autograd (forward of an x that requires gradients returns a
tensor without history): the caller passes x again and dx on.

PyTorch provides device memory and the stream only. Outputs and scratch are
allocated per call from torch's allocator on the current stream, so calls on
different streams and captured graphs do not share anything.
"""
from __future__ import annotations

from typing import Mapping

import torch

from . import prep
from . import weights as W
from .layers import TYPES, check_rows, entry, launch, workspace


def _in_place(m: torch.Tensor, stride: int) -> bool:
    """Whether the weight gradient reads this operand as it is (else through a bf16 copy in the workspace)."""
    return m.dtype == torch.bfloat16 and not (m.shape[1] | stride) & 1 and not m.data_ptr() & 3 and stride < 1 << 24


class BlockLinear:
    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, *, gradients: bool = False):
        """weight: e4m3 (torch.float8_e4m3fn, or its codes as uint8) [N, K] on the
        GPU; weight_scale: fp32 [ceil(N/128), ceil(K/128)]. Both are copied into
        the layer. gradients: also keep the layout input_gradient() reads."""
        if weight.dim() != 2 or weight.dtype not in (torch.float8_e4m3fn, torch.uint8) or not weight.is_cuda \
                or not weight.is_contiguous() or weight.numel() == 0:
            raise ValueError("BlockLinear needs a contiguous e4m3 (or uint8 codes) [N, K] GPU tensor")
        self.N, self.K = weight.shape
        grid = (-(-self.N // 128), -(-self.K // 128))
        if tuple(weight_scale.shape) != grid or weight_scale.dtype != torch.float32 or weight_scale.device != weight.device:
            raise ValueError(f"weight_scale: need torch.float32 {grid} on {weight.device}, got {weight_scale.dtype} "
                             f"{tuple(weight_scale.shape)} on {weight_scale.device}")
        self.device = weight.device
        self.scale = weight_scale.contiguous().clone()
        self._scale_ptr = self.scale.data_ptr()
        self._entries = {n: (entry(n), entry(n + "_workspace")) for n in (
            "netra_linear_forward", "netra_linear_input_gradient", "netra_linear_weight_gradient", "netra_linear_backward")}
        self.packed = self._pack(weight, 0)
        self.packed_t = self._pack(weight, 1) if gradients else None

    def _pack(self, weight: torch.Tensor, transpose: int) -> torch.Tensor:
        packed = torch.empty(entry("netra_linear_packed_bytes")(self.N, self.K, transpose), dtype=torch.uint8,
                             device=self.device)
        launch(entry("netra_linear_pack"), "netra_linear_pack", self.device, weight.data_ptr(), packed.data_ptr(), self.N, self.K, transpose)
        return packed

    @classmethod
    def from_float(cls, weight: torch.Tensor, *, gradients: bool = False) -> "BlockLinear":
        """Quantise fp32 [N, K] on the GPU per 128x128 block (netra_moe_quant_blocks'
        rule; short blocks are filled with zeros for it)."""
        if weight.dim() != 2 or weight.dtype != torch.float32 or not weight.is_cuda:
            raise ValueError("from_float needs an fp32 [N, K] GPU tensor")
        n, k = weight.shape
        full = torch.nn.functional.pad(weight, (0, -k % 128, 0, -n % 128)).contiguous()
        q, s = W.quantize_blocks(full[None])
        return cls(q[0, :n, :k].contiguous(), s[0], gradients=gradients)

    @classmethod
    def from_checkpoint(cls, tensors: Mapping[str, prep.TensorOrShards], name: str, device: torch.device, *,
                        gradients: bool = False) -> "BlockLinear":
        """{name}.weight (e4m3) and {name}.weight_scale_inv (bf16 or fp32), each a
        tensor or a list of output shards, host or device."""
        shards = prep._pieces(tensors, f"{name}.weight")
        n, k = sum(p.shape[0] for p in shards), shards[0].shape[1]
        if any(p.shape[0] % 128 for p in shards[:-1]):
            raise ValueError(f"{name}.weight: every output shard but the last needs a multiple of 128 rows")
        q = prep._weight(tensors, f"{name}.weight", n, k, device)
        s = prep._scale(tensors, f"{name}.weight_scale_inv", -(-n // 128), -(-k // 128), device)
        return cls(q, s, gradients=gradients)

    def _times(self, which: str, name: str, x: torch.Tensor, cols: int, out: torch.Tensor | None, out_cols: int,
               packed: torch.Tensor) -> torch.Tensor:
        rows = x.shape[0] if x.dim() == 2 else -1
        x_stride = check_rows(name, x, (rows, cols), self.device)
        if out is None:
            out, out_stride = torch.empty((rows, out_cols), dtype=torch.bfloat16, device=self.device), out_cols
        else:
            out_stride = check_rows("out", out, (rows, out_cols), self.device, (torch.bfloat16,))
        fn, need = self._entries[which]
        kind = TYPES[x.dtype]
        need = need(rows, self.N, self.K, kind)
        ws, ws_ptr = workspace(need, self.device)
        launch(fn, which, self.device, x.data_ptr(), kind, x_stride, packed.data_ptr(), self._scale_ptr,
               out.data_ptr(), out_stride, rows, self.N, self.K, ws_ptr, need)
        return out

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 or fp32 [T, K] -> x W^T, bf16 [T, N]."""
        return self._times("netra_linear_forward", "x", x, self.K, out, self.N, self.packed)

    __call__ = forward

    def input_gradient(self, dy: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """dy bf16 or fp32 [T, N] -> dy W, bf16 [T, K]."""
        if self.packed_t is None:
            raise ValueError("input_gradient needs a layer built with gradients=True")
        return self._times("netra_linear_input_gradient", "dy", dy, self.N, out, self.K, self.packed_t)

    def _weight_out(self, out: torch.Tensor | None, accumulate: bool) -> torch.Tensor:
        if out is None:
            if accumulate:
                raise ValueError("accumulate needs out")
            return torch.empty((self.N, self.K), dtype=torch.float32, device=self.device)
        if tuple(out.shape) != (self.N, self.K) or out.dtype != torch.float32 or not out.is_contiguous() \
                or out.device != self.device:
            raise ValueError(f"out: need contiguous torch.float32 {(self.N, self.K)} on {self.device}")
        return out

    def weight_gradient(self, dy: torch.Tensor, x: torch.Tensor, out: torch.Tensor | None = None, *,
                        accumulate: bool = False) -> torch.Tensor:
        """dy [T, N], x [T, K] -> dy^T x fp32 [N, K]; accumulate adds it to out."""
        rows = x.shape[0] if x.dim() == 2 else -1
        x_stride = check_rows("x", x, (rows, self.K), self.device)
        dy_stride = check_rows("dy", dy, (rows, self.N), self.device)
        out = self._weight_out(out, accumulate)
        name = "netra_linear_weight_gradient"
        fn, need = self._entries[name]
        need = need(rows, self.N, self.K, _in_place(x, x_stride) and _in_place(dy, dy_stride))
        ws, ws_ptr = workspace(need, self.device)
        launch(fn, name, self.device, dy.data_ptr(), TYPES[dy.dtype], dy_stride, x.data_ptr(), TYPES[x.dtype], x_stride,
               out.data_ptr(), int(accumulate), rows, self.N, self.K, ws_ptr, need)
        return out

    def backward(self, dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor | None = None, *,
                 accumulate: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
        """Both gradients: (dx, dw), as input_gradient() and weight_gradient() give them."""
        if self.packed_t is None:
            raise ValueError("backward needs a layer built with gradients=True")
        rows = x.shape[0] if x.dim() == 2 else -1
        x_stride = check_rows("x", x, (rows, self.K), self.device)
        dy_stride = check_rows("dy", dy, (rows, self.N), self.device)
        dw = self._weight_out(dw, accumulate)
        dx = torch.empty((rows, self.K), dtype=torch.bfloat16, device=self.device)
        name, kind = "netra_linear_backward", TYPES[dy.dtype]
        fn, need = self._entries[name]
        need = need(rows, self.N, self.K, kind, _in_place(x, x_stride) and _in_place(dy, dy_stride))
        ws, ws_ptr = workspace(need, self.device)
        launch(fn, name, self.device, dy.data_ptr(), kind, dy_stride, x.data_ptr(), TYPES[x.dtype], x_stride,
               self.packed_t.data_ptr(), self._scale_ptr, dx.data_ptr(), self.K, dw.data_ptr(), int(accumulate), rows,
               self.N, self.K, ws_ptr, need)
        return dx, dw
