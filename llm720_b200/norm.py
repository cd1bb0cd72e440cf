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

from . import _ext


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, checkpoint: Optional[str] = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's dtype.

    x is fp32, bf16 or fp16, of any shape and strides; weight and bias [D] are fp32 (what the reference keeps)
    or of x's dtype, and either may be missing.  ``checkpoint="e4m3"`` keeps x in 8 bits for the backward pass
    (a quarter to a half of the memory); y and the row statistics are those of the exact x.  Differentiable once,
    backward; a tensor with a forward-mode tangent is refused."""
    return _ext.load().layer_norm(x, weight, bias, eps, checkpoint)
