"""GPU parity of amdsplat.grad_norm, clip_grad_norm and FusedAdam.step(max_norm=...).

Bounds: the norm is a float64 sum rounded once (2^-24 relative, 2^-23 allowed); a clipped value is the
product with the once rounded coefficient (2^-24), rounded once to its type: 2^-23 in float32, 2^-8 +
2^-23 in bfloat16. The clipped Adam step is followed in float64 from the same state before each step: with
G = |g c|, m' and v' are two or three roundings from exact (2^-22 of the larger of old and new), and the
update lr m'/(sqrt(v') + eps), of three more operations, is off by 2^-21 of lr |m'| / sqrt(v') plus the
moments' own errors in it, and the parameter by one rounding. bfloat16 moments are rounded
stochastically, up to a whole unit in the last place (2^-7), before the update's float32 values are used
(the update itself takes the unrounded ones)."""
import math

import pytest
import torch

from amdsplat import FusedAdam, clip_grad_norm, grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def tensors(sizes, seed, mixed=True, scale=1.0, shift=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = (scale * torch.randn(n, generator=g)).to(torch.bfloat16 if mixed and i % 3 == 1 else torch.float32)
        if shift:  # addresses off every larger alignment
            buf = torch.empty(n + 1, dtype=t.dtype, device=DEV)
            buf[1:] = t.to(DEV)
            out.append(buf[1:])
        else:
            out.append(t.to(DEV))
    return out


def norm64(grads):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in grads))


SIZES = [
    [1], [2, 1], [7, 0, 5], [16384], [16385, 3], [100_003, 1, 64, 4096], [1] * 300, [5, 70_001] * 80,
    [0, 0, 3], list(range(1, 260)), [2_000_003, 12], [1 << 20] * 9,
]


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(sizes, shift):
    grads = tensors(sizes, len(sizes), shift=shift)
    want = norm64(grads)
    norm = grad_norm(grads)
    assert norm.dim() == 0 and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    for max_norm in (want / 3, want * 2):
        coef = min(1.0, max_norm / (want + 1e-6))
        keep = [t.clone() for t in grads]
        out = [torch.full_like(t, 7.0) for t in grads]
        got = clip_grad_norm(grads, max_norm, out=out)
        assert torch.equal(got, norm)
        for t, k, o in zip(grads, keep, out):
            assert torch.equal(t, k)
            off = (o.double() - k.double() * coef).abs()
            assert bool((off <= (2.0 ** -23 + UNIT[t.dtype]) * (k.double() * coef).abs()).all())
            if coef == 1.0:
                assert torch.equal(o, k)
        mine = [t.clone() for t in grads]
        assert torch.equal(clip_grad_norm(mine, max_norm), norm)
        assert all(torch.equal(a, b) for a, b in zip(mine, out))


def test_extremes():
    # squares beyond float32, squares below it
    for scale in (1e30, 1e-30):
        grads = tensors([5000, 77], 3, mixed=False, scale=scale)
        want = norm64(grads)
        assert abs(float(grad_norm(grads)) - want) <= 2.0 ** -23 * want
    zero = [torch.zeros(100, device=DEV)]
    assert float(clip_grad_norm(zero, 1.0)) == 0.0 and not bool(zero[0].any())
    assert float(grad_norm(torch.empty(0, device=DEV))) == 0.0
    one = [torch.ones(4, device=DEV)]
    clip_grad_norm(one, 0.0)
    assert not bool(one[0].any())
    bad = [torch.ones(4, device=DEV), torch.tensor([1.0, math.nan], device=DEV)]
    assert math.isnan(float(clip_grad_norm(bad, 1.0))) and bool(bad[0].isnan().all())
    inf = [torch.ones(4, device=DEV), torch.tensor([1.0, math.inf], device=DEV)]
    assert math.isinf(float(clip_grad_norm(inf, 1.0)))
    assert not bool(inf[0].any()) and float(inf[1][0]) == 0.0 and math.isnan(float(inf[1][1]))


def test_shapes_orders_and_bits():
    g = torch.Generator().manual_seed(4)
    a = torch.randn(37, 53, generator=g).to(DEV)
    assert torch.equal(grad_norm(a.t()), grad_norm(a.t().contiguous()))
    wide = torch.ones(1, device=DEV).expand(50)  # a broadcast gradient
    assert abs(float(grad_norm([wide])) - math.sqrt(50)) <= 1e-6
    assert torch.equal(grad_norm(iter([a, a])), grad_norm([a, a]))
    grads = tensors([100_000, 3, 50_000], 5)
    first = grad_norm(grads)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            again = grad_norm(grads)
        side.synchronize()
        assert torch.equal(first, again)


def test_agrees_with_torch():
    p = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (1000, 33, 4)]
    for x, t in zip(p, tensors([1000, 33, 4], 6, mixed=False)):
        x.grad = t
    mine = [x.grad.clone() for x in p]
    norm = clip_grad_norm(mine, 1.5)
    want = torch.nn.utils.clip_grad_norm_(p, 1.5)
    assert abs(float(norm) - float(want)) <= 1e-5 * float(want)
    for a, x in zip(mine, p):
        assert torch.allclose(a, x.grad, rtol=1e-5, atol=0)


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("loud", [False, True])
def test_clipped_adam_step(loud, sparse):
    n = 5003
    shapes = [(n, 3), (n, 3), (n, 4), (n, 1), (n, 1, 3), (n, 15, 3), (17, 5), (9,), (64, 64)]
    g = torch.Generator().manual_seed(7)
    vis = (torch.rand(n, generator=g) < 0.5).int().to(DEV)
    init = [torch.randn(*s, generator=g).to(DEV) for s in shapes]

    def optimizer():
        return FusedAdam([{"params": [torch.nn.Parameter(p.clone())], "lr": 1e-2, "name": str(i)}
                          for i, p in enumerate(init)], lr=0.0, eps=1e-15, sparse=sparse, lowp_moment_groups=("5",))

    opt = optimizer()
    mask = vis if sparse else None
    for step in range(1, 4):
        grads = [torch.randn(*s, generator=g).to(DEV) for s in shapes]
        want = norm64(grads)
        max_norm = want / 4 if loud else want * 4
        coef = min(1.0, max_norm / (want + 1e-6))
        before = []
        for grp, x in zip(opt.param_groups, grads):
            p = grp["params"][0]
            p.grad = x.clone()
            st = opt.state[p] if len(opt.state[p]) else None
            before.append([t.double() for t in (p.detach(), *((st["exp_avg"], st["exp_avg_sq"]) if st else
                                                              (torch.zeros_like(p), torch.zeros_like(p))))])
        norm = opt.step(visibility=mask, max_norm=max_norm)
        assert abs(float(norm) - want) <= 2.0 ** -23 * want
        for grp, x, (p0, m0, v0) in zip(opt.param_groups, grads, before):
            p = grp["params"][0]
            assert torch.equal(p.grad, x)
            c = x.double() * coef
            m, v = m0 + 0.1 * (c - m0), v0 + 0.001 * (c * c - v0)
            near_m, near_v = 2.0 ** -22 * torch.maximum(m0.abs(), c.abs()), 2.0 ** -22 * torch.maximum(v0, c * c)
            root = v.sqrt() / math.sqrt(1 - 0.999 ** step) + 1e-15
            lr = 1e-2 / (1 - 0.9 ** step)
            p1 = p0 - lr * m / root
            near_p = lr / root * (near_m + m.abs() * (near_v / v + 2.0 ** -21)) + 2.0 ** -23 * p1.abs()
            if mask is not None and p.shape[0] == n:
                hidden = (vis == 0)
                for t, t0 in ((p.detach(), p0), (opt.state[p]["exp_avg"], m0), (opt.state[p]["exp_avg_sq"], v0)):
                    assert torch.equal(t[hidden].double(), t0[hidden])
                live = (vis != 0)
            else:
                live = slice(None)
            low = 2.0 ** -7 if grp["name"] == "5" else 0.0
            for t, t1, near in ((p.detach(), p1, near_p), (opt.state[p]["exp_avg"], m, near_m + low * m.abs()),
                                (opt.state[p]["exp_avg_sq"], v, near_v + low * v)):
                assert bool(((t.double() - t1).abs() <= near)[live].all())


def test_refusals():
    t = torch.ones(10, device=DEV)
    for call, text in [
        (lambda: grad_norm([]), "no tensors"),
        (lambda: grad_norm([1.0]), "dense tensors"),
        (lambda: grad_norm([t.half()]), "float32 or bfloat16"),
        (lambda: grad_norm([t.cpu()]), "one GPU"),
        (lambda: grad_norm([t, t.cpu()]), "one GPU"),
        (lambda: clip_grad_norm([t], -1.0), "max_norm"),
        (lambda: clip_grad_norm([t], math.nan), "max_norm"),
        (lambda: clip_grad_norm([torch.ones(4, 5, device=DEV).t()], 1.0), "contiguous"),
        (lambda: clip_grad_norm([t], 1.0, out=[]), "no tensors"),
        (lambda: clip_grad_norm([t, t], 1.0, out=[t]), "outputs"),
        (lambda: clip_grad_norm([t], 1.0, out=[t[:9]]), "shapes"),
        (lambda: clip_grad_norm([t], 1.0, out=[t.bfloat16()]), "shapes"),
        (lambda: clip_grad_norm([t], 1.0, out=[torch.ones(5, 2, device=DEV).t()]), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    p = torch.nn.Parameter(t.clone())
    p.grad = torch.ones_like(p)
    opt = FusedAdam([{"params": [p], "lr": 1.0, "name": "p"}], lr=0.0, eps=1e-8)
    with pytest.raises(ValueError, match="max_norm"):
        opt.step(max_norm=-1.0)
    assert torch.equal(p.detach(), t) and len(opt.state[p]) == 0
