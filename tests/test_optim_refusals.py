"""A FusedAdam step that is refused leaves the optimizer as it was: no step is counted, no moment made."""
import pytest
import torch

from amdsplat import FusedAdam, adam


def optimizer(params, **kw):
    return FusedAdam([{"params": [p], "lr": 1e-2, "name": str(i)} for i, p in enumerate(params)], lr=0.0, eps=1e-8, **kw)


def refused(opt, text, **kw):
    before = {p: dict(s) for p, s in opt.state.items()}
    values = [g["params"][0].detach().clone() for g in opt.param_groups]
    with pytest.raises(ValueError, match=text):
        opt.step(**kw)
    after = {p: dict(s) for p, s in opt.state.items() if s}
    assert after.keys() == before.keys()
    for p, s in after.items():
        assert all(s[k] is before[p][k] or s[k] == before[p][k] for k in s), s
    assert all(torch.equal(g["params"][0].detach(), v) for g, v in zip(opt.param_groups, values))
    assert opt.n_dense_fallbacks == 0


def test_gradients_of_two_devices(monkeypatch):
    """The norm of gradients that are not on one GPU (the checks of the tensors themselves are left out, so that
    tensors of the CPU can stand for them)."""
    monkeypatch.setattr(adam, "_check", lambda *_: None)
    params = [torch.nn.Parameter(torch.ones(4, 3)) for _ in range(2)]
    for p in params:
        p.grad = torch.ones_like(p)
    refused(optimizer(params), "one GPU", max_norm=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, {"max_norm": 1.0}])
def test_the_last_parameter(kw):
    """A parameter that cannot be stepped behind one that can; then a visibility of another type."""
    good = torch.nn.Parameter(torch.ones(6, 3, device="cuda"))
    bad = torch.nn.Parameter(torch.ones(3, 6, device="cuda").t())
    good.grad, bad.grad = torch.ones_like(good), torch.ones_like(bad)
    opt = optimizer([good, bad], sparse=True)
    seen = torch.ones(6, dtype=torch.int32, device="cuda")
    refused(opt, "contiguous", visibility=seen, **kw)
    bad.grad = None
    opt.step(visibility=seen, **kw)
    assert opt.state[good]["step"] == 1 and not torch.equal(good.detach(), torch.ones_like(good))
    refused(opt, "int32", visibility=seen.long(), **kw)
    bad.grad = torch.ones_like(bad)
    refused(opt, "contiguous", visibility=seen, **kw)
    bad.grad = None
    opt.step(visibility=seen, **kw)
    assert opt.state[good]["step"] == 2
