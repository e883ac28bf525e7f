"""amdsplat.clip_grad_norm into other tensors and in place: which outputs it takes, and what autograd sees of its
writes."""
import pytest
import torch

from amdsplat import clip_grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_shapes_of_the_outputs():
    g = torch.randn(6, 10, generator=torch.Generator().manual_seed(0)).to(DEV)
    want = torch.empty_like(g)
    clip_grad_norm([g], 1.0, out=[want])
    flat = torch.empty(70, device=DEV)
    clip_grad_norm([g], 1.0, out=[flat[10:]])
    assert torch.equal(flat[10:].view(6, 10), want)
    # as many elements in another shape would take another order's values
    for shape in ((10, 6), (3, 20), (6, 10, 1), (59,), (61,)):
        with pytest.raises(ValueError, match="shapes"):
            clip_grad_norm([g], 1.0, out=[torch.empty(shape, device=DEV)])
