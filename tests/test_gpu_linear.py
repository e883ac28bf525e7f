"""GPU parity of amdsplat.linear against the formulas in float64.

Bounds. z is a float32 sum of K products and the bias: off by K 2^-24 of the sum of absolute values (its size). An
activation multiplies that by its slope (at most 1.2) and adds 2^-17 of its own value (the exponential's argument
z^2 / 2 up to 64 half-steps, a fit off by 1.6e-6). Then the sum with the residual and one rounding to the type, half a step: u =
2^-8 in bfloat16, 2^-24 in float32. Backward: dz is off by |dout| (c (z's error + u |z|) + 2^-16) + u |dz|, c the largest |act''|
(0.8 gelu, 0.5 silu; relu jumps where |z| is below its error), and the products by that times the other operand's absolute
values, by their length times 2^-24 of their size, and by one rounding."""
import math

import pytest
import torch

import block_ref as R
from amdsplat import linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def rand(seed, *shape, dtype=F32, gain=1.0):
    return (gain * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def inside(got, value, bound, what):
    off = (got.detach().double() - value).abs()
    bound = bound + UNIT[got.dtype] * value.abs() + 1e-37
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float((off / bound).max()))


def check(x, w, b=None, act="none", residual=None, train=True):
    leaves = {n: t.detach().requires_grad_(train) for n, t in (("x", x), ("weight", w), ("bias", b), ("residual", residual))
              if t is not None}
    (m, k), n = x.shape, w.shape[0]
    out = linear(**leaves, activation=act)
    assert out.shape == (m, n) and out.dtype == (x.dtype if residual is None else residual.dtype)
    d = rand(77, m, n, dtype=out.dtype) if train else None
    value, size = R.linear(x, w, b, act, residual, d)
    ez = (k + 2) * 2.0 ** -24 * size["z"]
    acted = value["out"] if residual is None else value["out"] - residual.double()
    rest = 0 if residual is None else residual.double().abs()
    e = (1.2 * ez + 2.0 ** -17 * acted.abs()) if act != "none" else ez
    inside(out, value["out"], e + 2.0 ** -23 * (acted.abs() + rest), "out")
    if not train:
        return out
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), d)))
    u = UNIT[x.dtype]
    edz = torch.zeros_like(value["dz"])
    if act != "none":
        edz = d.double().abs() * (R.CURVE[act] * (ez + u * value["z"].abs()) + 2.0 ** -16)
        if act == "relu":
            edz += d.double().abs() * (value["z"].abs() <= ez)
    unrounded = edz
    if act != "none" or out.dtype != x.dtype:
        edz = edz + u * value["dz"].abs()
    inside(grads["x"], value["d_x"], edz @ w.double().abs() + (n + 2) * 2.0 ** -24 * size["d_x"], "d_x")
    inside(grads["weight"], value["d_weight"], edz.t() @ x.double().abs() + (m + 2) * 2.0 ** -24 * size["d_weight"], "d_weight")
    if b is not None:
        assert grads["bias"].dtype == b.dtype
        inside(grads["bias"], value["d_bias"], unrounded.sum(0) + (m + 2) * 2.0 ** -24 * size["d_bias"], "d_bias")
    if residual is not None:
        assert torch.equal(grads["residual"], d)
    with torch.no_grad():
        again = linear(**leaves, activation=act)
    assert torch.equal(out, again)
    return out


def tensors(m, n, k, dtype, bias=F32, residual=None, seed=1):
    return (rand(seed, m, k, dtype=dtype), rand(seed + 1, n, k, dtype=dtype, gain=1 / math.sqrt(k)),
            None if bias is None else rand(seed + 2, n, dtype=bias),
            None if residual is None else rand(seed + 3, m, n, dtype=residual))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 8), (16, 17, 64), (33, 64, 65), (70, 130, 200)])
def test_forms(m, n, k, act, dtype):
    for bias in (None, F32, BF16):
        for residual in {None, F32, dtype}:
            x, w, b, r = tensors(m, n, k, dtype, bias, residual)
            check(x, w, b, act, r)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300])
def test_rows(m, dtype):
    for n, k in ((250, 576), (8, 24)):
        x, w, b, r = tensors(m, n, k, dtype, F32, F32)
        check(x, w, b, "silu", r)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 64, 65, 127, 255, 257, 513])
def test_outputs(n, dtype):
    for m, k in ((100, 72), (5, 300)):
        x, w, b, _ = tensors(m, n, k, dtype)
        check(x, w, b, "gelu")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [1, 2, 4, 7, 8, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 511, 577, 1000, 4096])
def test_inputs(k, dtype):
    for m, n in ((90, 72), (3, 40)):
        x, w, b, _ = tensors(m, n, k, dtype)
        check(x, w, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(2100, 4100, 200), (1030, 2050, 136), (4100, 257, 520), (257, 4100, 72), (9000, 40, 24), (40, 40, 9000)])
def test_large_tiles_and_splits(m, n, k, dtype):
    x, w, b, r = tensors(m, n, k, dtype, F32, dtype)
    check(x, w, b, "gelu", r)
    check(x, w, None, "none", None)


def test_no_rows():
    w, b = rand(1, 20, 24, dtype=BF16).requires_grad_(True), rand(2, 20).requires_grad_(True)
    x = torch.zeros(0, 24, dtype=BF16, device=DEV, requires_grad=True)
    out = linear(x, w, b, activation="gelu")
    assert out.shape == (0, 20)
    dx, dw, db = torch.autograd.grad(out.sum(), (x, w, b))
    assert dx.shape == (0, 24) and dw.eq(0).all() and db.eq(0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    big, wide = rand(1, 90, 200, dtype=dtype), rand(2, 70, 200, dtype=dtype, gain=0.1)
    b, r = rand(3, 140)[::2], rand(4, 90, 150, dtype=dtype)
    check(big[:, 16:112], wide[:, 8:104], b, "relu", r[:, 80:])
    check(big[::2, 16:112], wide[:, 8:104], b, "none", r[::2, 1:71])
    check(big[:, 1:97], wide[:, 3:99], None, "gelu", None)                     # addresses off: copied
    check(big[:, :96].t().contiguous().t(), wide[:, :96].t().contiguous().t())  # columns along: copied
    check(big[:1, :96].expand(90, 96), wide[:1, :96].expand(70, 96))           # one row for all
    check(big[:1, :96].expand(7, 96), wide[:, :96], None, "silu", r[:1, :70].expand(7, 70))
    odd = rand(5, 90, 101, dtype=dtype)
    check(odd[:, :96], wide[:, :96])                                           # a stride off: copied


def test_some_gradients():
    x, w, b, r = tensors(50, 60, 64, BF16, F32, F32)
    d = rand(9, 50, 60)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(linear(full[0], full[1], full[2], activation="gelu", residual=full[3]), full, d)
    for only in range(4):
        some = [t.clone().requires_grad_(i == only) for i, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(linear(some[0], some[1], some[2], activation="gelu", residual=some[3]), some[only], d)
        assert torch.equal(got, want[only])


def test_a_gradient_of_any_layout():
    """The output's gradient may be expanded, transposed or start at any address."""
    x, w, b, _ = tensors(50, 64, 64, BF16)
    for act in ("none", "gelu"):
        v = [t.clone().requires_grad_(True) for t in (x, w, b)]
        for d in (torch.ones(1, 1, dtype=BF16, device=DEV).expand(50, 64), rand(3, 64, 50, dtype=BF16).t(),
                  rand(4, 50 * 64 + 1, dtype=BF16)[1:].view(50, 64)):
            got = torch.autograd.grad(linear(*v, activation=act), v, d)
            want = torch.autograd.grad(linear(*v, activation=act), v, d.clone(memory_format=torch.contiguous_format))
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_activations_over_their_range():
    """One input per output, so that z is exact: tails to where they vanish, both types, infinities."""
    z = torch.cat((torch.linspace(-12, 12, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30]))).to(DEV)
    for dtype in (BF16, F32):
        x = z.to(dtype)[:, None].contiguous()
        one = torch.ones(1, 1, dtype=dtype, device=DEV)
        for act in ACTS:
            v = x.clone().requires_grad_(True)
            got = linear(v, one, activation=act, residual=torch.zeros(len(z), 1, device=DEV))
            want, slope = R.activate(x.double(), act)
            # the tail's exponent z^2 / 2 (72 at 12), or 1.6 (z + 0.045 z^3) of the tanh form (143), in half-steps
            inside(got, want, 2.0 ** -16 * want.abs(), act)
            # below 2^-126 (z under -12 in the tanh form) the hardware's exponential gives zero: 1e-37 is in the bound
            d, = torch.autograd.grad(got, v, torch.ones_like(got))
            inside(d, slope, 2.0 ** -16 * (slope.abs() + (x.double().abs() * want.abs())) + 2.0 ** -22, act)
    x = torch.tensor([[math.inf], [-math.inf], [math.nan]], device=DEV)
    one = torch.ones(1, 1, device=DEV)
    assert linear(x, one, activation="relu").flatten().tolist()[:2] == [math.inf, 0.0]
    for act in ACTS:
        y = linear(x, one, activation=act).flatten()
        assert y[0] == math.inf and bool(torch.isnan(y[2]))


def test_what_is_not_finite_stays_in_its_row_and_column():
    x, w, b, _ = tensors(300, 200, 128, BF16)
    want = linear(x, w, b, activation="gelu")
    x2, w2 = x.clone(), w.clone()
    x2[70, 3], w2[130, 5] = math.inf, math.nan
    got = linear(x2, w2, b, activation="gelu")
    rows, cols = [i for i in range(300) if i != 70], [i for i in range(200) if i != 130]
    assert torch.equal(got[rows][:, cols], want[rows][:, cols])
    assert bool(torch.isnan(got[:, 130]).all())
    # few rows, whose other rows and columns hold the same
    few, spoiled = linear(x[64:75], w, b, activation="gelu"), linear(x2[64:75], w2, b, activation="gelu")
    rows = [i for i in range(11) if i != 6]
    assert torch.equal(spoiled[rows][:, cols], few[rows][:, cols]) and bool(torch.isnan(spoiled[:, 130]).all())
    # memory behind the tensors is not read into results
    big = torch.full((40, 128), math.nan, dtype=BF16, device=DEV)
    big[:33, :72] = x[:33, :72]
    weights = torch.full((60, 128), math.nan, dtype=BF16, device=DEV)
    weights[:50, :72] = w[:50, :72]
    for m in (5, 33):
        check(big[:m, :72], weights[:50, :72], None, "silu")


def test_gradient_against_differences():
    """Without an activation linear in x, so a difference of any step is the directional derivative; float32."""
    x, w, b, _ = tensors(80, 72, 96, F32)
    way, d = rand(5, 80, 96), rand(6, 80, 72)
    x.requires_grad_(True)
    g, = torch.autograd.grad(linear(x, w, b), x, d)
    with torch.no_grad():
        slope = float(((linear(x + way, w, b).double() - linear(x, w, b).double()) * d.double()).sum())
        mine = float((g.double() * way.double()).sum())
        size = (2 * x.abs() + way.abs()).double() @ w.double().abs().t() + 2 * b.double().abs()
        room = float(((98 + 74 + 2) * 2.0 ** -24 * size * d.double().abs()).sum())
    assert abs(mine - slope) <= room


def test_captured_with_its_backward():
    x, w, b, r = (t.requires_grad_(True) for t in tensors(200, 136, 264, BF16, F32, F32))
    d = rand(8, 200, 136)

    def step():
        out = linear(x, w, b, activation="gelu", residual=r)
        return out.detach(), *torch.autograd.grad(out, (x, w, b, r), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        with torch.no_grad():
            x.copy_(rand(seed, 200, 264, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_on_a_side_stream():
    x, w, b, _ = tensors(500, 512, 1024, BF16)
    want = linear(x, w, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = linear(x, w, b)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    x, w = z(4, 16), z(8, 16)
    for args, kw, text in [
        ((z(4), w), {}, "must be"), ((x, z(8, 15)), {}, "must be"), ((x.half(), w.half()), {}, "dtype"),
        ((x, w.float()), {}, "dtype"), ((x, w.cpu()), {}, "GPU"), ((x, z(0, 16)), {}, "outputs"), ((z(4, 0), z(8, 0)), {}, "inputs"),
        ((x, w, z(7)), {}, "bias must"), ((x, w, z(8).half()), {}, "bias must"), ((x, w), dict(residual=z(4, 7)), "residual must"),
        ((x, w), dict(residual=z(4, 8).half()), "residual must"),
        ((x.float(), w.float()), dict(residual=z(4, 8)), "residual must"), ((x, w), dict(activation="tanh"), "activation must"),
    ]:
        with pytest.raises(ValueError, match=text):
            linear(*args, **kw)
