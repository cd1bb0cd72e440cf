"""Activation checkpoints in 8 bits.

What a training step keeps of an activation between its forward and its
backward pass takes two (four) bytes a value; in row-scaled e4m3 it takes one.
A row ``x`` is stored as bytes ``p`` and one fp32 scale ``s``: the smallest power of
two with ``max|x| / s <= 448`` over the row's finite values (1 for a row of
zeros, never below 2^-126), ``p = e4m3(x / s)`` to nearest even.  ``p * s`` differs
from ``x`` by at most 2^-4 of ``|x|`` (of ``2^-6 s`` below that value).  Infinite
and NaN values become NaN.

``layer_norm(..., checkpoint="e4m3")`` and ``PEER.activation_checkpoint = "e4m3"``
keep their inputs in this form by themselves; the two functions here are for a
program's own autograd functions.
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import _ext


def pack_rows_e4m3(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., D] (fp32, bf16 or fp16) -> (payload float8_e4m3fn [..., D], scale fp32 [...]).  Not differentiable."""
    return _ext.load().pack_rows(x)


def unpack_rows_e4m3(payload: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``pack_rows_e4m3``'s result stands for, clamped to the finite range of ``dtype``
    (scale may be any fp32 numbers).  Not differentiable."""
    return _ext.load().unpack_rows(payload, scale, dtype)
