"""ctypes binding of the operators next to the MoE layer (include/netra_layers.h,
libnetra_layers.so), and what their Python forms share."""
from __future__ import annotations

import ctypes

import torch

from . import paths

P, U32, U64, F32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float

# entry point -> (result, arguments)
SIGNATURES = {
    "netra_linear_packed_bytes": (U64, [U32] * 3),
    "netra_linear_pack": (ctypes.c_int, [P, P, U32, U32, U32, P]),
    "netra_linear_forward_workspace": (U64, [U32] * 3),
    "netra_linear_input_gradient_workspace": (U64, [U32] * 3),
    "netra_linear_weight_gradient_workspace": (U64, [U32] * 3),
    "netra_linear_forward": (ctypes.c_int, [P, U32, U64, P, P, P, U64, U32, U32, U32, P, U64, P]),
    "netra_linear_input_gradient": (ctypes.c_int, [P, U32, U64, P, P, P, U64, U32, U32, U32, P, U64, P]),
    "netra_linear_weight_gradient": (ctypes.c_int, [P, U32, U64, P, U32, U64, P, U32, U32, U32, U32, P, U64, P]),
    "netra_router_counts_workspace": (U64, [U32] * 3),
    "netra_router_counts": (ctypes.c_int, [P, U64, P, U32, U32, U32, P, U32, P, U64, P]),
    "netra_router_balance_workspace": (U64, [U32] * 3),
    "netra_router_balance": (ctypes.c_int, [P, U32, U64, P, P, U64, U32, P, U32, U32, F32, P, P, P, U64, P, U64, P]),
    "netra_layers_last_error": (ctypes.c_char_p, []),
}
TYPES = {torch.bfloat16: 0, torch.float32: 1}  # NETRA_BF16, NETRA_F32

_lib = None


def library() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        path = paths.layers_library()
        if not path.is_file():
            raise FileNotFoundError(f"{path} is missing: build the native library first")
        lib = ctypes.CDLL(str(path))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def call(name: str, device: torch.device, *args) -> None:
    """Launch one entry point on the device's current stream; raises on a nonzero status."""
    lib = library()
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        rc = getattr(lib, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, stream)
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {(lib.netra_layers_last_error() or b'').decode()}")


def check_rows(name: str, t: torch.Tensor, shape: tuple[int, int], device: torch.device, dtypes=tuple(TYPES)) -> None:
    """A matrix with unit column stride and rows that do not overlap, on the device."""
    if (t.dim() != 2 or tuple(t.shape) != shape or t.dtype not in dtypes or t.device != device
            or (t.stride(1) != 1 and shape[1] > 1) or (t.stride(0) < shape[1] and shape[0] > 1)):
        raise ValueError(f"{name}: need {' or '.join(map(str, dtypes))} {shape} on {device} with contiguous rows, got "
                         f"{t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}")


def row_stride(t: torch.Tensor) -> int:
    """Row stride in elements (of a single row: its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]
