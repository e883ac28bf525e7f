"""The block operators together, as the predictor example runs them: its fused blocks against the same model with plain
torch operations in their place, in training and with cached scenes. float32; both sides are float32 sums in other
orders through a few layers, whose gradients are compared to 1e-3 of their size."""
import importlib.util
import sys
from pathlib import Path

import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parent.parent / "3dgs-project_amd" / "examples" / "predict_splats.py"
    spec = importlib.util.spec_from_file_location("predict_splats", path)
    module = importlib.util.module_from_spec(spec)
    sys.modules["predict_splats"] = module
    spec.loader.exec_module(module)
    return module


def plain_norm(x, weight=None, bias=None, *, kind="rms", eps=1e-6, dtype=None):
    return x * (x.square().mean(1, keepdim=True) + eps) ** -0.5 * weight


def plain_residual_norm(x, y, weight, *, post_weight=None, gate=None, dropout=0.0, seed=None, draw=0):
    b = y if post_weight is None else plain_norm(y, post_weight)
    if dropout:
        b = b * R.keep(*y.shape, int(seed), draw, dropout).float().to(y.device)
    h = x + (b if gate is None else gate * b)
    return h, plain_norm(h, weight)


def plain_linear(x, weight, bias=None, *, activation="none", residual=None):
    z = torch.nn.functional.linear(x, weight, bias)
    z = torch.nn.functional.gelu(z) if activation == "gelu" else z
    return z if residual is None else z + residual


def plain_scan(x, forget, gate, *, offsets=None, initial=None, return_state=False):
    cuts = [0, x.shape[0]] if offsets is None else offsets.tolist()
    a, ys, states = torch.sigmoid(forget), [], []
    for d in range(len(cuts) - 1):
        h = torch.zeros_like(x[0]) if initial is None else initial[d]
        for t in range(cuts[d], cuts[d + 1]):
            h = a[t] * h + (1 - a[t]) * x[t]
            ys.append(h * torch.nn.functional.silu(gate[t]))
        states.append(h)
    y = torch.stack(ys)
    return (y, torch.stack(states)) if return_state else y


def plainly(E, monkeypatch):
    for name, f in (("norm", plain_norm), ("residual_norm", plain_residual_norm), ("linear", plain_linear),
                    ("gated_scan", plain_scan)):
        monkeypatch.setattr(E, name, f)


def config(E, **kw):
    return E.Config(image=32, width=64, depth=2, heads=2, kv_heads=1, dtype=torch.float32, **kw)


FORMS = [dict(), dict(sandwich=True, dropout=0.2), dict(scan=(1,)), dict(sandwich=True, dropout=0.1, scan=(0,))]


@pytest.mark.parametrize("form", FORMS)
def test_training_step_against_plain_operations(form, monkeypatch):
    E = example()
    c = config(E, fused=True, **form)
    scenes = [E.synthetic_scene(i, 2 + i, c.image, n=100) for i in range(2)]

    def run():
        model = E.SplatPredictor(c)
        out = model(scenes)
        g = torch.Generator().manual_seed(3)
        total = sum((t * torch.randn(t.shape, generator=g).to(t.device)).sum() for o in out for t in o.values())
        names, ps = zip(*model.named_parameters())
        return out, dict(zip(names, torch.autograd.grad(total, ps)))

    out, grads = run()
    plainly(E, monkeypatch)
    want, want_grads = run()
    for a, b in zip(out, want):
        for name in a:
            assert torch.allclose(a[name], b[name], rtol=1e-4, atol=1e-4), name
    for name, g in grads.items():
        off, size = float((g - want_grads[name]).norm()), float(want_grads[name].norm())
        assert size > 0 and off <= 1e-3 * size, (name, off / size)


def test_fused_blocks_are_the_plain_model():
    """The same weights through the composed and the fused blocks."""
    E = example()
    scenes = [E.synthetic_scene(i, 2 + i, 32, n=100) for i in range(2)]
    with torch.no_grad():
        a, b = (E.SplatPredictor(config(E, fused=f))(scenes) for f in (False, True))
    for x, y in zip(a, b):
        for name in x:
            assert torch.allclose(x[name], y[name], rtol=1e-4, atol=1e-4), name


@pytest.mark.parametrize("form", [dict(scan=(0, 1)), dict(sandwich=True, scan=(0, 1))])
def test_added_views_continue_the_recurrence(form):
    """Layers that mix in order give a view that is added later what it would have had in the packed scene."""
    E = example()
    c = config(E, fused=True, **form)
    model = E.SplatPredictor(c).eval()
    images, cams = E.synthetic_scene(5, 4, c.image, n=100)
    cache = model.cache(images[:2], cams[:2], room=200)
    got = [model.extend(cache, images[i], cams[i]) for i in (2, 3)]
    with torch.no_grad():
        want = model([(images, cams)])[0]
    n = got[0]["means"].shape[0]
    for i, g in enumerate(got):
        for name in g:
            assert torch.allclose(g[name], want[name][(2 + i) * n:(3 + i) * n], rtol=1e-4, atol=1e-4), name


def test_steps_in_bfloat16():
    E = example()
    c = E.Config(image=32, width=64, depth=2, heads=2, kv_heads=1, fused=True, sandwich=True, dropout=0.1, scan=(1,))
    model = E.SplatPredictor(c)
    optimizer = E.optimizer_for(model)
    scenes = [E.synthetic_scene(i, 2 + i, c.image, n=100) for i in range(2)]
    first = int(model.seed)
    for _ in range(3):
        loss, norm = E.train_step(model, optimizer, scenes)
        assert bool(torch.isfinite(loss)) and float(norm) > 0
    assert int(model.seed) == first + 3
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and bool(p.grad.any()) for p in model.parameters())
    model.eval()
    images, cams = scenes[1]
    cache = model.cache(images[:2], cams[:2], room=100)
    assert bool(torch.isfinite(model.extend(cache, images[2], cams[2])["means"]).all())


def test_a_captured_block_with_its_backward():
    """norm, projection, recurrence, projection, residual norm and MLP in one graph, forward and backward, replayed on other
    inputs and another seed against eager runs."""
    from amdsplat import gated_scan, linear, norm, residual_norm

    g = torch.Generator().manual_seed(1)
    r = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    w = [(0.1 * r(n, k, dtype=torch.bfloat16)).requires_grad_(True) for n, k in ((360, 96), (96, 120), (384, 96), (96, 384))]
    v = [(1 + 0.1 * r(96)).requires_grad_(True) for _ in range(4)]
    x, offsets = r(150, 96).requires_grad_(True), torch.tensor([0, 50, 50, 150], dtype=torch.int32, device="cuda")
    seed, d = torch.tensor([5], device="cuda"), r(150, 96)

    def step():
        n = norm(x, v[0], dtype=torch.bfloat16)
        y = linear(gated_scan(*linear(n, w[0]).chunk(3, 1), offsets=offsets), w[1])
        h, n = residual_norm(x, y, v[1], post_weight=v[2], gate=v[3], dropout=0.1, seed=seed)
        h = linear(linear(n, w[2], activation="silu"), w[3], residual=h)
        return h.detach(), *torch.autograd.grad(h, (x, *w, *v), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(r(150, 96))
            seed.fill_(7 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
