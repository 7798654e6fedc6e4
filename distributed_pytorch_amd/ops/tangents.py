"""Which calls have to go through an operator's autograd function.

An operator that nobody differentiates may call its kernels directly.  A gradient being recorded is one reason not to; a
forward-mode tangent (``torch.autograd.forward_ad``) is the other, although such a tensor does not require gradients:
the kernels would drop the tangent without a word, the autograd function raises.

The reference's operators are torch's own (reference min_DDP.py:44-49), which take both kinds of derivative.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad


def is_differentiated(*tensors: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level < 0:  # (outside of any dual level no tensor has a tangent; looked at first, for single tokens wait for the host)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
