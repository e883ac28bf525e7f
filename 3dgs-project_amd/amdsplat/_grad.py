"""What calls of operators do about derivatives that they do not provide."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def tracked(*tensors) -> bool:
    """An input takes a gradient, or a forward-mode level is entered, where an input may carry a tangent: the
    functions have no forward-mode derivative and say so, while reading the input's data alone would drop it."""
    return forward_ad._current_level >= 0 or (
        torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def refuse_tangents(tensors, what: str) -> None:
    """For calls without any derivative: a tangent is refused."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: no forward-mode derivative")
