"""The block operators where offsets pass 2^31 elements, and their refusal of forward-mode tangents. Values at the far end
are compared with the same call on the far rows alone, bit by bit: a row's result does not depend on the others."""
import pytest
import torch
from torch.autograd import forward_ad

import block_ref as R
from amdsplat import dropout, gated_scan, linear, norm, residual_norm

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda", torch.bfloat16


def rand(seed, *shape, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def test_far_rows_of_a_projection():
    """2.2e9 results, and gradients of as many."""
    m, k, n = 530_003, 64, 4096
    x, w, b = rand(1, m, k), rand(2, n, k), rand(3, n, dtype=torch.float32)
    out = linear(x, w, b, activation="relu")
    for rows in (slice(0, 300), slice(m - 300, m)):
        assert torch.equal(out[rows], linear(x[rows], w, b, activation="relu"))
    del out
    x.requires_grad_(True)
    wide = rand(4, n, m // 8, dtype=BF16)  # and where a row of the weight is long
    y = rand(5, 40, m // 8)
    far = linear(y, wide)
    value, size = R.linear(y, wide)
    assert bool(((far.double() - value["out"]).abs() <= 2.0 ** -8 * value["out"].abs() + (m // 8) * 2.0 ** -24 * size["z"]).all())
    d = rand(6, m, n)
    dx, = torch.autograd.grad(linear(x, w), x, d)
    rows = slice(m - 300, m)
    near = x[rows].detach().requires_grad_(True)
    want, = torch.autograd.grad(linear(near, w), near, d[rows])
    assert torch.allclose(dx[rows].float(), want.float(), rtol=2.0 ** -7, atol=1e-2)


def test_far_rows_of_norms_and_dropout():
    t, c = 2_100_001, 1024
    x, y, w = rand(1, t, c), rand(2, t, c), rand(3, c, dtype=torch.float32)
    rows = slice(t - 100, t)
    h, n = residual_norm(x, y, w, post_weight=w)
    want = residual_norm(x[rows], y[rows], w, post_weight=w)
    assert torch.equal(h[rows], want[0]) and torch.equal(n[rows], want[1])
    del h, n
    xs = x.requires_grad_(True)
    dx, = torch.autograd.grad(norm(xs, w), xs, y)
    near = x[rows].detach().requires_grad_(True)
    assert torch.equal(dx[rows], torch.autograd.grad(norm(near, w), near, y[rows])[0])
    del dx
    out = dropout(x.detach(), 0.25, 9)
    # a row's bits go by its number: rows of the whole against the generator's
    k = R.keep(4, c, 9, 0, 0.25)
    assert torch.equal(out[:4] == 0, (k == 0).to(DEV) | (x[:4] == 0))
    last = [t - 1, t - 77]
    for r in last:
        words = [R.philox([g, r, 0, 0], [9, 0]) for g in range(c // 8)]
        bits = torch.tensor([h for four in words for word in four for h in (word & 0xffff, word >> 16)])
        dropped = (bits < 16384).to(DEV) | (x[r] == 0)
        assert torch.equal(out[r] == 0, dropped)


def test_far_tokens_of_a_recurrence():
    t, c = 2_100_001, 1024
    x, f = rand(1, t, c), rand(2, t, c)
    cut = t - 333
    offsets = torch.tensor([0, cut, t], dtype=torch.int32, device=DEV)
    y, state = gated_scan(x, f, offsets=offsets, return_state=True)
    value, size = R.gated_scan(x[cut:].cpu(), f[cut:].cpu())
    off = (y[cut:].double().cpu() - value["y"]).abs()
    assert bool((off <= 2.0 ** -15 * size["y"] + 2.0 ** -8 * value["y"].abs()).all())
    assert bool(((state[1].double().cpu() - value["state"][0]).abs() <= 2.0 ** -15 * size["state"][0]).all())
    d = rand(3, t, c)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(gated_scan(x, f, offsets=offsets), x, d)
    value, size = R.gated_scan(x[cut:].detach().cpu(), f[cut:].cpu(), d_y=d[cut:].cpu())
    off = (dx[cut:].double().cpu() - value["d_x"]).abs()
    assert bool((off <= 2.0 ** -15 * size["d_x"] + 2.0 ** -8 * value["d_x"].abs()).all())


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    x, w, v = rand(1, 20, 64, dtype=torch.float32), rand(2, 48, 64, dtype=torch.float32), rand(3, 64, dtype=torch.float32)
    calls = {
        "linear": lambda a: linear(a, w), "weight": lambda a: linear(x, a[:16]), "norm": lambda a: norm(a, v),
        "residual": lambda a: residual_norm(x, a, v), "dropout": lambda a: dropout(a, 0.5, 1), "scan": lambda a: gated_scan(x, a),
    }
    plain = {n: f(x) for n, f in calls.items()}
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f in calls.values():
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                f(dual)
        for n, f in calls.items():  # without a tangent the level changes nothing
            a, b = (t if isinstance(t, tuple) else (t,) for t in (f(x), plain[n]))
            assert all(torch.equal(p, q) for p, q in zip(a, b))
