"""The gradient norm and clipping have no derivative: a forward-mode tangent is refused (before the check for the
GPU, so that the CPU shows it)."""
import pytest
import torch
from torch.autograd import forward_ad

from amdsplat import clip_grad_norm, grad_norm


def test_tangents_are_refused():
    x = torch.randn(5)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(5))
        for call in (lambda: grad_norm(dual), lambda: grad_norm([x, dual]), lambda: clip_grad_norm([dual], 1.0)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="GPU"):
            grad_norm([x])
