"""Scaled embedding lookup with a gradient that is summed by sorted tokens.

The reference's model reads its token table with ``nn.Embedding``
(llm/models/foundation.py:338).  Here the lookup multiplies by a constant in the
same pass, and the backward pass sorts the token positions by id and adds every
id's rows in fp32 in a fixed order: the gradient does not vary from run to run,
whatever the ids' frequencies are.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._rows import as_rows, launch, require_cuda, require_dtype

_MAX_ROWS = 2**31 - 2


def _lookup(ids, weight, scale, dropped, dt):
    out = torch.empty(ids.shape + weight.shape[1:], dtype=weight.dtype, device=weight.device)
    launch(_lib.load().peer_embedding, weight.device, ids.data_ptr(), ids.element_size(), ids.numel(), weight.data_ptr(), dt,
           *weight.shape, scale, out.data_ptr(), None if dropped is None else dropped.data_ptr())
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, dropped, dt):
        ctx.save_for_backward(ids)
        ctx.args = (scale, padding_idx, dt, weight.shape)
        return _lookup(ids, weight, scale, dropped, dt)

    @staticmethod
    def backward(ctx, grad_out):
        return _embedding_grad_once(ctx, grad_out) if torch.is_grad_enabled() else _embedding_grad(ctx, grad_out)


def _embedding_grad(ctx, grad_out):
    ids, = ctx.saved_tensors
    scale, padding_idx, dt, (V, D) = ctx.args
    rows = as_rows(grad_out)
    dev = grad_out.device
    lib = _lib.load()
    n = ids.numel()
    grad = torch.empty(V, D, dtype=grad_out.dtype, device=dev)
    nbytes = lib.peer_embedding_workspace(n, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    launch(lib.peer_embedding_backward, dev, ids.data_ptr(), ids.element_size(), n, rows.data_ptr(), rows.stride(0), dt, V, D,
           scale, -1 if padding_idx is None else padding_idx, grad.data_ptr(), ws.data_ptr(), nbytes)
    return grad, None, None, None, None, None


_embedding_grad_once = once_differentiable(_embedding_grad)     # create_graph=True: a second derivative raises


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, *, padding_idx: Optional[int] = None,
              dropped: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * weight[ids]``: ids int32 or int64 of any shape, weight [V, D] fp32, bf16 or fp16.

    An id outside [0, V) (-1 for a position without a token, say) reads nothing: its row is zero and takes no
    part in the gradient; ``dropped`` (int64 [1] on the device) is increased by the number of such ids.  The row
    ``padding_idx`` is read like any other and receives a gradient of zero.  Differentiable once, in weight."""
    require_cuda(weight, "weight")
    dt = require_dtype(weight, "weight")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be a [rows, width] table, got {tuple(weight.shape)}")
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids is {ids.dtype}, expected int32 or int64")
    if ids.device != weight.device:
        raise RuntimeError(f"ids is on {ids.device}, weight on {weight.device}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx={padding_idx} of a table of {weight.shape[0]} rows")
    if dropped is not None and (dropped.dtype != torch.int64 or dropped.numel() != 1 or dropped.device != weight.device):
        raise TypeError("dropped must be one int64 on the table's device")
    if ids.numel() > _MAX_ROWS or weight.shape[0] > _MAX_ROWS:
        raise ValueError("more than 2^31 - 2 ids or table rows")
    ids = ids.contiguous()
    scale = float(scale)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(weight, ids, scale, padding_idx, dropped, dt)
    return _lookup(ids, weight, scale, dropped, dt)
