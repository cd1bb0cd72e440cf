"""Layer norm with a gradient: the ``ln_2`` in front of the layer (reference:
llm/models/foundation.py:118, 196-199) for training.

``PEER.block_forward`` has the norm built in but is an inference path; this is
the same norm as a differentiable operator, with an option to keep its input for
the backward pass in 8 bits (``checkpoint="e4m3"``, the format of
``checkpoint.pack_rows_e4m3``).  The gradient of the weight and the bias is summed
in fp32 in a fixed order, so it does not vary from run to run.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._rows import as_rows, launch, require_cuda, require_dtype


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def norm_forward(x: torch.Tensor, weight, bias, eps: float, dt: int, pdt: int, keep: bool, pack: bool):
    """(y, stats, payload, scale): y of x's shape; with ``keep`` the rows' means and 1/deviations as stats [2, rows],
    with ``pack`` x in 8 bits, else None."""
    rows = as_rows(x)
    R, D = rows.shape
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = payload = scale = mean = rstd = None
    if keep:
        stats = torch.empty(2, R, dtype=torch.float32, device=dev)
        mean = stats.data_ptr()
        rstd = mean + 4 * R
    if pack:
        payload = torch.empty(R, D, dtype=torch.float8_e4m3fn, device=dev)
        scale = torch.empty(R, dtype=torch.float32, device=dev)
    launch(_lib.load().peer_layer_norm, dev, rows.data_ptr(), rows.stride(0), dt, _ptr(weight), _ptr(bias), pdt, eps, R, D,
           y.data_ptr(), mean, rstd, _ptr(payload), _ptr(scale))
    return y, stats, payload, scale


def norm_backward(grad_y: torch.Tensor, x, payload, scale, stats, weight, dt: int, pdt: int, want_x: bool, weight_dtype,
                  bias_dtype, add: Optional[torch.Tensor] = None):
    """(dx, dweight, dbias); ``weight_dtype`` / ``bias_dtype`` None: that sum is not wanted.  x or its packed form.
    ``add`` (contiguous, of x's shape) is added to dx before its rounding."""
    grad_rows = as_rows(grad_y)
    R, D = grad_rows.shape
    dev = grad_y.device
    lib = _lib.load()
    rows = None if x is None else as_rows(x)
    dx = torch.empty(grad_y.shape, dtype=grad_y.dtype, device=dev) if want_x else None
    dw = None if weight_dtype is None else torch.empty(D, dtype=weight_dtype, device=dev)
    db = None if bias_dtype is None else torch.empty(D, dtype=bias_dtype, device=dev)
    ws, nbytes = None, 0
    if dw is not None or db is not None:
        nbytes = lib.peer_layer_norm_workspace(R, D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    mean = stats.data_ptr()
    launch(lib.peer_layer_norm_backward, dev, grad_rows.data_ptr(), grad_rows.stride(0), _ptr(rows),
           0 if rows is None else rows.stride(0), _ptr(payload), _ptr(scale), mean, mean + 4 * R, _ptr(weight), dt, pdt, _ptr(add),
           R, D, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint, dt, pdt):
        packed = checkpoint == "e4m3"
        y, stats, payload, scale = norm_forward(x, weight, bias, eps, dt, pdt, True, packed)
        ctx.save_for_backward(None if packed else x, weight, payload, scale, stats)
        ctx.codes = (dt, pdt)
        ctx.param_dtypes = (None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        return _norm_grad_once(ctx, grad_y) if torch.is_grad_enabled() else _norm_grad(ctx, grad_y)


def _norm_grad(ctx, grad_y):
    x, weight, payload, scale, stats = ctx.saved_tensors
    want_x, want_w, want_b = ctx.needs_input_grad[:3]
    wdt, bdt = ctx.param_dtypes
    dx, dw, db = norm_backward(grad_y, x, payload, scale, stats, weight, *ctx.codes, want_x, wdt if want_w else None,
                               bdt if want_b else None)
    return dx, dw, db, None, None, None, None


_norm_grad_once = once_differentiable(_norm_grad)     # create_graph=True: a second derivative raises


def check_norm_arguments(x, weight, bias, eps):
    """Raise on what the kernels do not take; (dtype code of x, of the parameters)."""
    require_cuda(x, "x")
    dt = require_dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one value, got shape {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps={eps} must not be negative")
    pdt = _lib.DTYPE_F32
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{name} is {tuple(p.shape)}, expected ({x.shape[-1]},)")
        if p.device != x.device:
            raise RuntimeError(f"{name} is on {p.device}, x on {x.device}")
        if p.dtype != torch.float32 and p.dtype != x.dtype:
            raise TypeError(f"{name} is {p.dtype}: parameters are float32 or of x's dtype, {x.dtype}")
        if not p.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        pdt = require_dtype(p, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: both parameters have one dtype")
    return dt, pdt


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, checkpoint: Optional[str] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's dtype.

    x is fp32, bf16 or fp16, of any shape and strides; weight and bias [D] are fp32 (what the reference keeps)
    or of x's dtype, and either may be missing.  ``checkpoint="e4m3"`` keeps x in 8 bits for the backward pass
    (a quarter to a half of the memory); y and the row statistics are those of the exact x.  Differentiable once."""
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"checkpoint={checkpoint!r}: None or 'e4m3'")
    dt, pdt = check_norm_arguments(x, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, checkpoint, dt, pdt)
    return norm_forward(x, weight, bias, eps, dt, pdt, False, False)[0]
