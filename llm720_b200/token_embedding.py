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

from . import _ext


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, *, padding_idx: Optional[int] = None,
              dropped: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * weight[ids]``: ids int32 or int64 of any shape, weight [V, D] fp32, bf16 or fp16.

    An id outside [0, V) (-1 for a position without a token, say) reads nothing: its row is zero and takes no
    part in the gradient; ``dropped`` (int64 [1] on the device) is increased by the number of such ids.  The row
    ``padding_idx`` is read like any other and receives a gradient of zero.  Differentiable once, backward, in
    weight; a table with a forward-mode tangent is refused."""
    return _ext.load().embedding(ids, weight, scale, padding_idx, dropped)
