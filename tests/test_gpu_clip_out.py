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


def test_autograd_sees_the_writes():
    """A tensor saved for a backward pass and clipped in between: the pass raises, as after any other write."""
    for into in (False, True):
        g = torch.randn(20, device=DEV)
        x = torch.ones(20, device=DEV, requires_grad=True)
        out = [torch.empty(20, device=DEV)] if into else None
        written = out[0] if into else g
        before, other = written._version, (g if into else x)._version
        y = (x * written).sum()
        clip_grad_norm([g], 1e-3, out=out)
        assert written._version > before and (g if into else x)._version == other
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        g = torch.randn(20, device=DEV)
        clip_grad_norm([g], 1e-3)
        assert float(g.norm()) < 2e-3
