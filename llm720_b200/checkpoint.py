"""Activation checkpoints in 8 bits.

What a training step keeps of an activation between its forward and its
backward pass takes two (four) bytes a value; in row-scaled e4m3 it takes one.
A row ``x`` is stored as bytes ``p`` and one fp32 scale ``s``: the smallest power
of two with ``max|x| / s <= 448`` over the row's finite values (1 for a row of
zeros, never below 2^-126), ``p = e4m3(x / s)`` to nearest even.  ``p * s`` differs
from ``x`` by at most 2^-4 of ``|x|`` (of ``2^-6 s`` below that value).  Infinite
and NaN values become NaN.

``layer_norm(..., checkpoint="e4m3")`` and ``PEER.block_train`` keep their inputs
in this form by themselves; the two functions here are for a program's own
autograd functions.
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import _lib
from ._rows import DTYPES, as_rows, launch, require_cuda, require_dtype


def pack_rows_e4m3(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., D] (fp32, bf16 or fp16) -> (payload float8_e4m3fn [..., D], scale fp32 [...]).  Not differentiable."""
    require_cuda(x, "x")
    dt = require_dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one value, got shape {tuple(x.shape)}")
    x = x.detach()
    payload = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rows = as_rows(x)
    launch(_lib.load().peer_pack_rows, x.device, rows.data_ptr(), rows.stride(0), dt, *rows.shape, payload.data_ptr(),
           scale.data_ptr())
    return payload, scale


def unpack_rows_e4m3(payload: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``pack_rows_e4m3``'s result stands for, clamped to the finite range of ``dtype``."""
    require_cuda(payload, "payload")
    if payload.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        raise TypeError(f"payload is {payload.dtype} and scale {scale.dtype}, expected float8_e4m3fn and float32")
    if dtype not in DTYPES:
        raise TypeError(f"dtype {dtype}: float32, bfloat16 and float16 are implemented")
    if payload.dim() < 1 or payload.shape[-1] < 1 or scale.shape != payload.shape[:-1]:
        raise ValueError(f"payload {tuple(payload.shape)} and scale {tuple(scale.shape)} do not belong together")
    if scale.device != payload.device:
        raise RuntimeError(f"scale is on {scale.device}, payload on {payload.device}")
    payload, scale = payload.contiguous(), scale.contiguous()
    out = torch.empty(payload.shape, dtype=dtype, device=payload.device)
    D = payload.shape[-1]
    launch(_lib.load().peer_unpack_rows, payload.device, payload.data_ptr(), scale.data_ptr(), DTYPES[dtype],
           payload.numel() // D, D, out.data_ptr())
    return out
