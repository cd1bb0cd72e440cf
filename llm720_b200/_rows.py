"""Argument handling shared by the row-wise operators (``layer_norm``,
``pack_rows_e4m3``, ``embedding``): what the C entry points take is a matrix of
rows of consecutive values with one row stride."""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def require_cuda(t: torch.Tensor, name: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} is on {t.device}: peer_b200 runs on CUDA devices only (sm_100a); there is no CPU path")


def require_dtype(t: torch.Tensor, name: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} is {t.dtype}; float32, bfloat16 and float16 are implemented")
    return code


def as_rows(t: torch.Tensor) -> torch.Tensor:
    """t [..., D] as [rows, D] with consecutive values in a row: a view wherever one exists (row strides of any
    size, zero included, are the kernels' business), else a contiguous copy."""
    D = t.shape[-1]
    rows = t if t.dim() == 2 else t.reshape(-1, D) if t.numel() else t.reshape(t.numel() // D, D)
    return rows if D == 1 or rows.stride(1) == 1 else rows.contiguous()


# torch.cuda.current_stream and torch.cuda.device cost 4 and 1.5 us a call, more than the launch they are for; the raw
# accessors cost 0.2 us
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def launch(entry, device: torch.device, *args) -> None:
    """Call a C entry point with the current stream of ``device`` as its last argument; raise on an error code."""
    index = device.index
    if _current_device() == index:
        rc = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)
