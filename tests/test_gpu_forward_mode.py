"""Forward-mode derivatives of the predictor's operators: there are none, and a tangent is not dropped without a
word."""
import pytest
import torch
from torch.autograd import forward_ad

from amdsplat import attention, rotary_axes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tangents_are_refused(dtype, grad):
    x = torch.randn(20, 2, 64, device="cuda").to(dtype)
    pos = torch.arange(20.0, device="cuda")[:, None]
    plain = attention(x, x, x), rotary_axes(x, None, pos, (16,))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: attention(dual, x, x), lambda: attention(x, dual, x), lambda: attention(x, x, dual),
                     lambda: attention(dual[..., :30], x[..., :30], x[..., :30]),
                     lambda: rotary_axes(dual, None, pos, (16,)), lambda: rotary_axes(x, dual, pos, (16,))):
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                call()
        # without a tangent the level changes nothing
        again = attention(x, x, x), rotary_axes(x, None, pos, (16,))
    for a, b in zip(plain, again):
        assert torch.equal(a, b)
