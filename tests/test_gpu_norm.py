"""GPU parity of amdsplat.norm, residual_norm and dropout against the formulas in float64.

Bound of a float32 evaluation: a standardised row is a difference, scaled by a deviation whose square is a sum of at
most 32 terms a lane and six to ten steps across lanes, so it is off by at most 2^-18 of its size (the formula with
absolute values), and what two norms, products and row means build on it by 2^-16 of theirs. A column sum
adds at most 2^-17 of its own for the rows of a workgroup and the join. Then one rounding to the type: half a step,
2^-8 of the value in bfloat16, 2^-24 in float32. Dropout alone is one product: its factor's rounding and the
result's."""
import math

import pytest
import torch

import block_ref as R
from amdsplat import dropout, norm, residual_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


def rand(seed, *shape, dtype=F32, gain=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (gain * torch.randn(shape, generator=g) + shift).to(dtype).to(DEV)


def near(got, value, size, what):
    off = (got.detach().double().cpu() - value.cpu()).abs()
    bound = 2.0 ** -16 * size.cpu() + UNIT[got.dtype] * value.cpu().abs() + 1e-37
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float((off / bound).max()))


def check(x, y, w, b, pw, pb, gate, kind, scale, p, draw=5, seed=1234567890123, eps=1e-6):
    leaves = dict(x=x, y=y, weight=w, bias=b, post_weight=pw, post_bias=pb, gate=gate)
    leaves = {n: t.detach().requires_grad_(True) for n, t in leaves.items() if t is not None}
    t, c = x.shape
    d_h, d_n = rand(901, t, c, dtype=x.dtype), rand(902, t, c, dtype=y.dtype)
    h, n = residual_norm(**leaves, kind=kind, eps=eps, scale=scale, dropout=p, seed=seed, draw=draw)
    assert h.dtype == x.dtype and n.dtype == y.dtype
    grads = dict(zip(leaves, torch.autograd.grad((h, n), list(leaves.values()), (d_h, d_n))))
    factors = R.keep(t, c, seed, draw, p).to(DEV) if p else None
    value, size = R.residual_norm(**leaves, kind=kind, eps=eps, scale=scale, factors=factors, d_h=d_h, d_n=d_n)
    near(h, value["h"], size["h"], "h")
    near(n, value["n"], size["n"], "n")
    for name, g in grads.items():
        assert g.shape == leaves[name].shape and g.dtype == leaves[name].dtype
        near(g, value["d_" + name], size["d_" + name], "d_" + name)
    with torch.no_grad():
        h2, n2 = residual_norm(**leaves, kind=kind, eps=eps, scale=scale, dropout=p, seed=seed, draw=draw)
    assert torch.equal(h, h2) and torch.equal(n, n2)


@pytest.mark.parametrize("stream,branch", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", [None, "column", "token"])
def test_forms(stream, branch, kind, gate):
    for t, c, post, p in ((1, 1, False, 0.0), (3, 7, True, 0.0), (5, 64, True, 0.4), (70, 130, False, 0.2), (9, 513, True, 0.1)):
        v = lambda s: rand(s, c, gain=0.3, shift=1.0)  # noqa: E731
        g = {None: None, "column": v(5), "token": rand(5, t, c, dtype=branch)}[gate]
        layer = kind == "layer"
        check(rand(1, t, c, dtype=stream, gain=2, shift=0.5), rand(2, t, c, dtype=branch), v(3), v(4) if layer else None,
              v(6) if post else None, v(7) if post and layer else None, g, kind, 0.7, p)


@pytest.mark.parametrize("width", [1, 2, 8, 63, 512, 520, 645, 1024, 1025, 2048, 2050, 4096, 5000, 8191, 8192])
def test_widths(width):
    stream, branch = TYPES[width % 3]
    v = lambda s: rand(s, width, gain=0.3, shift=1.0)  # noqa: E731
    check(rand(1, 6, width, dtype=stream), rand(2, 6, width, dtype=branch), v(3), v(4), v(6), v(7), v(8), "layer", 1.0, 0.3)


@pytest.mark.parametrize("rows", [1, 2, 5, 511, 2049, 4099])
def test_lengths(rows):
    v = lambda s: rand(s, 250, gain=0.3, shift=1.0)  # noqa: E731
    check(rand(1, rows, 250), rand(2, rows, 250, dtype=BF16), v(3), None, v(6), None, v(7), "rms", 1.0, 0.1)


def test_no_rows_and_plain_norm():
    z = torch.zeros(0, 40, device=DEV, requires_grad=True)
    w = torch.ones(40, device=DEV, requires_grad=True)
    h, n = residual_norm(z, z.detach(), w)
    dw, = torch.autograd.grad((h.sum() + n.sum()), w)
    assert h.shape == n.shape == (0, 40) and torch.equal(dw, torch.zeros_like(w))
    for dtype, to in ((F32, F32), (F32, BF16), (BF16, BF16)):
        for kind in ("rms", "layer"):
            x, w, b = rand(1, 37, 100, dtype=dtype, shift=1).requires_grad_(True), rand(2, 100).requires_grad_(True), rand(3, 100).requires_grad_(True)
            d = rand(4, 37, 100, dtype=to)
            got = norm(x, w, b, kind=kind, dtype=to)
            assert got.dtype == to
            value, size = R.residual_norm(x, None, w, b, kind=kind, d_n=d)
            near(got, value["n"], size["n"], "n")
            for g, name in zip(torch.autograd.grad(got, (x, w, b), d), ("d_x", "d_weight", "d_bias")):
                near(g, value[name], size[name], name)
            near(norm(x, kind=kind, dtype=to), *(r["n"] for r in R.residual_norm(x, None, kind=kind)), "no weight")


@pytest.mark.parametrize("stream,branch", TYPES)
@pytest.mark.parametrize("width", [4104, 6001])
@pytest.mark.parametrize("rows", [3, 1100])
def test_wide_rows(rows, width, stream, branch):
    """Above 4096 columns the backward keeps its column sums elsewhere: all five, some and none of them, rows than which there
    are fewer workgroups."""
    v = lambda s: rand(s, width, gain=0.3, shift=1.0)  # noqa: E731
    x, y = rand(1, rows, width, dtype=stream), rand(2, rows, width, dtype=branch)
    check(x, y, v(3), v(4), v(5), v(6), v(7), "layer", 0.5, 0.1)
    if rows == 3:
        check(x, y, None, v(4), v(5), None, rand(8, rows, width), "rms", 1.0, 0.0)
        check(x, y, None, None, None, None, v(7), "rms", 1.0, 0.3)
        check(x, y, None, None, None, None, None, "layer", 1.0, 0.0)


def test_one_of_the_gradients():
    """Only h or only n goes on, only some inputs take a gradient, weights in bfloat16."""
    x, y = rand(1, 20, 96).requires_grad_(True), rand(2, 20, 96, dtype=BF16)
    w = rand(3, 96, dtype=BF16).requires_grad_(True)
    pw = rand(4, 96, dtype=BF16)
    d_h, d_n = rand(5, 20, 96), rand(6, 20, 96, dtype=BF16)
    for through_h, through_n in ((True, False), (False, True)):
        h, n = residual_norm(x, y, w, post_weight=pw)
        given = dict(d_h=d_h if through_h else None, d_n=d_n if through_n else None)
        value, size = R.residual_norm(x, y, w, post_weight=pw, **given)
        out, d = (h, d_h) if through_h else (n, d_n)
        gx, gw = torch.autograd.grad(out, (x, w), d)
        near(gx, value["d_x"], size["d_x"], "d_x")
        near(gw, value["d_weight"], size["d_weight"], "d_weight")


def test_strides_and_rows_of_a_wider_tensor():
    big = rand(1, 50, 3 * 77 + 5)
    low = big.to(BF16)
    for x, y, g in ((big[:, 1:78], low[:, 80:157], low[:, 3:80]), (big[::2, :77], low[::2, 5:82], big[::2, 78:155]),
                    (big[:, :77], low[:1, :77].expand(50, 77), low[:1, 9:86].expand(50, 77)),
                    (big[:, :77].t().contiguous().t(), low[:, :77], None)):
        check(x, y, rand(2, 154)[::2], None, rand(3, 77), None, g, "rms", 0.5, 0.2)


def test_loud_and_constant_rows():
    """Rows around a large mean lose nothing but what float32 inputs lose; a zero row's norm is zero."""
    x = rand(1, 8, 200, shift=1000.0)
    value, size = R.residual_norm(x, None, kind="layer")
    near(norm(x, kind="layer"), value["n"], size["n"], "n")
    z = torch.zeros(3, 200, device=DEV)
    for kind in ("rms", "layer"):
        assert norm(z, kind=kind).eq(0).all() and norm(z + 3, kind="layer").eq(0).all()
    # 2^-20 of values of 2^40, and values whose squares leave float32's normal numbers
    for gain in (2.0 ** 40, 2.0 ** 60, 2.0 ** -60):
        check(rand(1, 4, 130, gain=gain), rand(2, 4, 130, gain=gain), rand(3, 130), None, rand(4, 130), None, None, "rms",
              1.0, 0.0, eps=1e-30)


def test_what_is_not_finite_stays_in_its_row():
    x, y, w = rand(1, 9, 64), rand(2, 9, 64), rand(3, 64)
    want = residual_norm(x, y, w, post_weight=w)
    x2, y2 = x.clone(), y.clone()
    x2[2, 5], y2[7, 1] = math.inf, math.nan
    got = residual_norm(x2, y2, w, post_weight=w)
    keep = [0, 1, 3, 4, 5, 6, 8]
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])
    # a dropped element is zero whatever it was (no post norm)
    k = R.keep(9, 64, 5, 0, 0.5).to(DEV) == 0
    bad = torch.where(k, torch.full_like(y, math.nan), y)
    for a, b in zip(residual_norm(x, bad, w, dropout=0.5, seed=5), residual_norm(x, y, w, dropout=0.5, seed=5)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 8), (33, 250), (3, 5, 77), (2049, 64), (4, 0), (0, 9)])
def test_dropout(shape, dtype):
    x = rand(1, *shape, dtype=dtype).requires_grad_(True)
    width = shape[-1]
    rows = math.prod(shape[:-1])
    for p, seed, draw in ((0.0, None, 0), (0.1, 5, 0), (0.5, (1 << 62) + 12345, (1 << 40) + 7), (0.99999, -3, 1)):
        out = dropout(x, p, seed, draw=draw)
        k = (R.keep(rows, width, (seed or 0) % (1 << 64), draw, p) if p else torch.ones(rows, width, dtype=torch.float64)).reshape(shape)
        value = x.detach().double().cpu() * k
        assert bool(((out.detach().double().cpu() - value).abs() <= (2 * UNIT[F32] + UNIT[dtype]) * value.abs()).all())
        d = rand(2, *shape, dtype=dtype)
        g, = torch.autograd.grad(out, x, d)
        value = d.double().cpu() * k
        assert bool(((g.double().cpu() - value).abs() <= (2 * UNIT[F32] + UNIT[dtype]) * value.abs()).all())


def test_dropout_seeds():
    x = torch.ones(300, 160, device=DEV)
    at = torch.tensor([77], dtype=torch.int64, device=DEV)
    a = dropout(x, 0.25, 77, draw=3)
    assert torch.equal(a, dropout(x, 0.25, at, draw=3))
    assert not torch.equal(a, dropout(x, 0.25, 78, draw=3)) and not torch.equal(a, dropout(x, 0.25, 77, draw=4))
    # a binomial count of 48000 elements: six deviations are 570
    assert abs(int((a == 0).sum()) - 12000) < 570
    assert torch.equal(a, dropout(torch.ones(300, 161, device=DEV)[:, :160], 0.25, 77, draw=3))
    bad = torch.where(a == 0, torch.full_like(x, math.nan), x)
    assert torch.equal(dropout(bad, 0.25, 77, draw=3), a)
    # written between forward and backward: the mask of the forward is gone, and autograd says so
    y = x.clone().requires_grad_(True)
    out = dropout(y, 0.25, at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_replayed_with_other_seeds():
    """A captured training step whose seed advances inside the graph, against eager runs."""
    x, y, w = rand(1, 64, 96).requires_grad_(True), rand(2, 64, 96, dtype=BF16).requires_grad_(True), rand(3, 96).requires_grad_(True)
    d_h, d_n = rand(4, 64, 96), rand(5, 64, 96, dtype=BF16)
    seed = torch.tensor([10], dtype=torch.int64, device=DEV)

    def step():
        h, n = residual_norm(x, y, w, gate=w.detach(), dropout=0.3, seed=seed, draw=1)
        return h.detach(), n.detach(), *torch.autograd.grad((h, n), (x, y, w), (d_h, d_n))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for value in (10, 11, 12, 11):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_on_a_side_stream():
    x, y, w = rand(1, 300, 512), rand(2, 300, 512, dtype=BF16), rand(3, 512)
    want = residual_norm(x, y, w, dropout=0.1, seed=3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = residual_norm(x, y, w, dropout=0.1, seed=3)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    x, y, w = z(4, 8), z(4, 8), z(8)
    for args, kw, text in [
        ((x, z(4, 9), w), {}, "alike"), ((z(4), z(4), w), {}, "alike"), ((x, y.cpu(), w), {}, "GPU"),
        ((x.half(), y.half(), w), {}, "float32 or bfloat16"), ((x.bfloat16(), y, w), {}, "does not go with"),
        ((x, y.half(), w), {}, "does not go with"), ((x, y, z(9)), {}, "weight must be"), ((x, y, w.half()), {}, "weight must be"),
        ((x, y, w, z(8, dtype=BF16)), {}, "bias must be"), ((x, y, w), dict(post_bias=w), "without post_weight"),
        ((x, y, w), dict(post_weight=w.cpu()), "post_weight must be"), ((x, y, w), dict(gate=z(4)), "gate must be"),
        ((x, y, w), dict(gate=z(8, dtype=torch.int32)), "gate must be"), ((x, y, w), dict(kind="batch"), "kind"),
        ((x, y, w), dict(eps=0.0), "eps"), ((x, y, w), dict(eps=math.nan), "eps"), ((x, y, w), dict(scale=math.inf), "scale"),
        ((x, y, w), dict(dropout=1.0, seed=1), "probability"), ((x, y, w), dict(dropout=0.5), "seed"),
        ((x, y, w), dict(dropout=0.5, seed=torch.zeros(1, dtype=torch.int64)), "seed"),
        ((x, y, w), dict(dropout=0.5, seed=1 << 64), "64 bits"), ((x, y, w), dict(dropout=0.5, seed=1, draw=-1), "draw"),
        ((z(2, 8193), z(2, 8193)), {}, "width"), ((z(2, 0), z(2, 0)), {}, "width"),
    ]:
        with pytest.raises(ValueError, match=text):
            residual_norm(*args, **kw)
    with pytest.raises(ValueError, match="does not go with"):
        norm(x, dtype=torch.float16)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        dropout(x.half(), 0.5, 1)
