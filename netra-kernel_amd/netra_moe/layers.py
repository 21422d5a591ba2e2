"""ctypes binding of the operators next to the MoE layer (include/netra_layers.h,
libnetra_layers.so), and what their Python forms share."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import paths

P, U32, U64, F32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float

# entry point -> (result, arguments)
SIGNATURES = {
    "netra_linear_packed_bytes": (U64, [U32] * 3),
    "netra_linear_pack": (ctypes.c_int, [P, P, U32, U32, U32, P]),
    "netra_linear_forward_workspace": (U64, [U32] * 4),
    "netra_linear_input_gradient_workspace": (U64, [U32] * 4),
    "netra_linear_weight_gradient_workspace": (U64, [U32] * 4),
    "netra_linear_forward": (ctypes.c_int, [P, U32, U64, P, P, P, U64, U32, U32, U32, P, U64, P]),
    "netra_linear_forward_codes_workspace": (U64, [U32] * 3),
    "netra_linear_forward_codes": (ctypes.c_int, [P, P, P, P, P, U64, U32, U32, U32, P, U64, P]),
    "netra_linear_input_gradient": (ctypes.c_int, [P, U32, U64, P, P, P, U64, U32, U32, U32, P, U64, P]),
    "netra_linear_weight_gradient": (ctypes.c_int, [P, U32, U64, P, U32, U64, P, U32, U32, U32, U32, P, U64, P]),
    "netra_linear_backward_workspace": (U64, [U32] * 5),
    "netra_linear_backward": (ctypes.c_int, [P, U32, U64, P, U32, U64, P, P, P, U64, P, U32, U32, U32, U32, P, U64, P]),
    "netra_router_counts_workspace": (U64, [U32] * 3),
    "netra_router_counts": (ctypes.c_int, [P, U64, P, U32, U32, U32, P, U32, P, U64, P]),
    "netra_router_balance_workspace": (U64, [U32] * 3),
    "netra_router_balance": (ctypes.c_int, [P, U32, U64, P, P, U64, U32, P, U32, U32, F32, P, P, P, U64, P, U64, P]),
    "netra_norm_code_bytes": (U64, [U32] * 3),
    "netra_norm_scale_count": (U64, [U32] * 3),
    "netra_norm_forward": (ctypes.c_int, [P, U32, U64, P, U32, U64, P, U32, F32, F32, P, U64, P, U32, U64, P, P, U32, U32, U32, P]),
    "netra_norm_gradients_workspace": (U64, [U32] * 2),
    "netra_norm_gradients": (ctypes.c_int, [P, U32, U64, P, U32, U64, P, U64, P, U32, F32, F32, P, U64, P, U32, U32, U32, P, U64, P]),
    "netra_router_select": (ctypes.c_int, [P, U32, U64, P, P] + [U32] * 9 + [F32, P, U64, P, U64, P]),
    "netra_router_select_gradient": (ctypes.c_int, [P, U64, P, U32, U64, P, U64, P] + [U32] * 6 + [F32, P, U64, U32, P]),
    "netra_adapters_packed_bytes": (U64, [U32] * 5),
    "netra_adapters_pack": (ctypes.c_int, [P, P, U32, P, P] + [U32] * 4 + [P]),
    "netra_adapters_plan_bytes": (U64, [U32] * 2),
    "netra_adapters_plan": (ctypes.c_int, [P, U32, U32, P, U64, P]),
    "netra_adapters_add_workspace": (U64, [U32] * 5),
    "netra_adapters_add": (ctypes.c_int, [P, U32, U64, P, P, P, P, P, U64, P, U64] + [U32] * 5 + [P, U64, P]),
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


@functools.lru_cache(maxsize=None)
def entry(name: str):
    """An entry point as a plain callable, looked up once."""
    return getattr(library(), name)


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(d).cuda_stream without the object (1.8 us a call)


def launch(fn, name: str, device: torch.device, *args) -> None:
    """Launch an entry point on the device's current stream; raises on a nonzero status."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {(library().netra_layers_last_error() or b'').decode()}")


def workspace(need: int, device: torch.device) -> tuple[torch.Tensor | None, int]:
    """Scratch of one call from torch's allocator (the tensor keeps it alive over the launch), and its address."""
    if not need:
        return None, 0
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def check_rows(name: str, t: torch.Tensor, shape: tuple[int, int], device: torch.device, dtypes=TYPES) -> int:
    """A matrix with unit column stride and rows that do not overlap, on the device.
    Returns its row stride in elements (of a single row: its length)."""
    if t.shape == shape and t.dtype in dtypes and t.device == device:
        rows, cols = t.stride()
        if (cols == 1 or shape[1] <= 1) and (rows >= shape[1] or shape[0] <= 1):
            return rows if shape[0] > 1 else shape[1]
    raise ValueError(f"{name}: need {' or '.join(map(str, dtypes))} {shape} on {device} with contiguous rows, got "
                     f"{t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}")
