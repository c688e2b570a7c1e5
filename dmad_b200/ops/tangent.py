"""Forward-mode derivatives: how operators that have none notice one."""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwd


def carries_tangent(*tensors) -> bool:
    """Whether one of ``tensors`` (None allowed) is a dual tensor of the current forward-mode level.  A dual tensor
    requires no gradient, so a kernel called on its memory would drop the tangent without a sign."""
    if fwd._current_level < 0 or not torch._C._is_fwd_grad_enabled():
        return False
    return any(t is not None and fwd.unpack_dual(t).tangent is not None for t in tensors)
