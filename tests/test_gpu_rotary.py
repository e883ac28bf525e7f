"""GPU parity of amdsplat.rotary_axes against the formula in float64.

Bound: the angle is off by at most 2^-23 turns' worth of float32 rounding and cos and sin by an ulp,
2^-22 in all, so an element of a turned pair (u, w) is off by 2^-22 (|u| + |w|) and one rounding to the
type (2^-8 of it in bfloat16, 2^-24 in float32)."""
import math

import pytest
import torch

from amdsplat import rotary_axes

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DT = [torch.bfloat16, torch.float32]


def formula(x, positions, sections, base, pairing, spectrum, inverse=False):
    x, positions = x.double().cpu(), positions.double().cpu()
    pairs = sum(sections)
    y, bound = x.clone(), torch.zeros_like(x)
    p = 0
    for axis, n in enumerate(sections):
        for j in range(n):
            freq = base ** -(p / pairs if spectrum == "shared" else j / n)
            angle = positions[:, axis] * freq * (-1 if inverse else 1)
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            a, b = (p, p + pairs) if pairing == "half" else (2 * p, 2 * p + 1)
            u, w = x[..., a], x[..., b]
            y[..., a], y[..., b] = u * c - w * s, u * s + w * c
            bound[..., a] = bound[..., b] = 2.0 ** -22 * (u.abs() + w.abs())
            p += 1
    return y, bound


def check(got, want):
    value, bound = want
    bound = bound + UNIT[got.dtype] * value.abs()
    off = (got.detach().cpu().double() - value).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def data(tokens, heads, dim, dtype, seed, axes, span=200.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    return x.to(DEV), (span * torch.rand(tokens, axes, generator=g)).to(DEV)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("spectrum", ["axis", "shared"])
@pytest.mark.parametrize("dim,sections", [(64, (10, 11, 11)), (64, (32,)), (72, (15, 16)), (40, (4, 4, 4, 8)),
                                          (2, (1,)), (7, (1, 2)), (128, (16, 24, 24)), (96, (16, 16)),
                                          (80, (0, 8, 8)), (33, (5, 3))])
def test_forward_and_gradient(dim, sections, pairing, spectrum, dtype):
    for tokens, heads, kv in ((1, 3, 1), (37, 4, 2), (130, 1, 5)):
        q, pos = data(tokens, heads, dim, dtype, tokens, len(sections))
        k, _ = data(tokens, kv, dim, dtype, tokens + 1, len(sections))
        gq, _ = data(tokens, heads, dim, dtype, tokens + 2, len(sections))
        gk, _ = data(tokens, kv, dim, dtype, tokens + 3, len(sections))
        q.requires_grad_(True), k.requires_grad_(True)
        rule = (sections, 10000.0, pairing, spectrum)
        q2, k2 = rotary_axes(q, k, pos, sections, pairing=pairing, spectrum=spectrum)
        dq, dk = torch.autograd.grad((q2, k2), (q, k), (gq, gk))
        for got, x, inverse in ((q2, q, False), (k2, k, False), (dq, gq, True), (dk, gk, True)):
            assert got.dtype == dtype and got.shape == x.shape
            check(got, formula(x.detach(), pos, *rule, inverse=inverse))


@pytest.mark.parametrize("dtype", DT)
def test_strides_alignment_and_one_tensor(dtype):
    g = torch.Generator().manual_seed(5)
    for dim in (64, 33):
        rows = torch.randn(90, 11, dim + 1, generator=g).to(dtype).to(DEV)
        pos = (20 * torch.rand(90, 2, generator=g)).to(DEV)
        views = [rows[:, :4, :dim], rows[:, 4:, 1:], rows[:, ::2, :dim], rows[::3, :4, 1:],
                 rows[:, :4, :dim].permute(2, 0, 1).contiguous().permute(1, 2, 0),
                 rows[:, :1, :dim].expand(90, 6, dim)]
        for x in views:
            at = pos[:x.shape[0]]
            got = rotary_axes(x, None, at, (7, 9), base=500.0)
            check(got, formula(x, at, (7, 9), 500.0, "half", "axis"))
            two = rotary_axes(x, rows[:x.shape[0], :2, :dim], at, (7, 9), base=500.0, pairing="adjacent")
            check(two[0], formula(x, at, (7, 9), 500.0, "adjacent", "axis"))
            check(two[1], formula(rows[:x.shape[0], :2, :dim], at, (7, 9), 500.0, "adjacent", "axis"))


def test_positions_of_every_kind():
    x, _ = data(50, 2, 64, torch.float32, 6, 1)
    g = torch.Generator().manual_seed(7)
    grid = torch.randint(-300, 300, (50, 2), generator=g)
    for pos in (grid.to(DEV), grid.int().to(DEV), grid.short().to(DEV), grid.float().to(DEV),
                grid.t().contiguous().to(DEV).t()):
        check(rotary_axes(x, None, pos, (16, 16)), formula(x, grid, (16, 16), 10000.0, "half", "axis"))
    # far positions: the angle is reduced before it is rounded
    far = torch.randint(0, 1 << 24, (50, 2), generator=g).float()
    check(rotary_axes(x, None, far.to(DEV), (16, 16)), formula(x, far, (16, 16), 10000.0, "half", "axis"))


@pytest.mark.parametrize("tokens", [0, 1, 4099])
def test_lengths(tokens):
    q, pos = data(tokens, 16, 64, torch.bfloat16, 8, 3)
    k, _ = data(tokens, 16, 64, torch.bfloat16, 9, 3)
    a, b = rotary_axes(q, k, pos, (8, 12, 12))
    check(a, formula(q, pos, (8, 12, 12), 10000.0, "half", "axis"))
    check(b, formula(k, pos, (8, 12, 12), 10000.0, "half", "axis"))


def test_gradient_against_differences():
    """The operator is linear in x, so a difference of any step is its directional derivative:
    float32, step 1, tolerance of the two forwards' and the gradient's rounding."""
    x, pos = data(40, 3, 64, torch.float32, 10, 2)
    w, _ = data(40, 3, 64, torch.float32, 11, 2)
    way, _ = data(40, 3, 64, torch.float32, 12, 2)
    x.requires_grad_(True)
    grad, = torch.autograd.grad(rotary_axes(x, None, pos, (10, 12)), x, w)
    with torch.no_grad():
        up, down = rotary_axes(x + way, None, pos, (10, 12)), rotary_axes(x, None, pos, (10, 12))
        slope = float(((up.double() - down.double()) * w.double()).sum())
        mine = float((grad.double() * way.double()).sum())
        size = float(((x.abs() + way.abs()).double() * w.abs().double()).sum())
    assert abs(mine - slope) <= 8 * 2.0 ** -22 * size * math.sqrt(2)


def test_on_a_side_stream():
    q, pos = data(500, 8, 64, torch.bfloat16, 13, 2)
    want = rotary_axes(q, None, pos, (16, 16))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rotary_axes(q, None, pos, (16, 16))
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    q, pos = z(10, 4, 64), z(10, 2, dtype=torch.float32)
    for args, kw, text in [
        ((z(10, 64), None, pos, (4, 4)), {}, "tokens, heads"),
        ((q.half(), None, pos, (4, 4)), {}, "dtype"),
        ((q, z(10, 2, 64, dtype=torch.float32), pos, (4, 4)), {}, "dtype"),
        ((q, None, pos.cpu(), (4, 4)), {}, "GPU"),
        ((q, z(9, 2, 64), pos, (4, 4)), {}, "shape mismatch"),
        ((q, z(10, 0, 64), pos, (4, 4)), {}, "head"),
        ((q, None, pos, ()), {}, "sections"),
        ((q, None, pos, (4, -1)), {}, "sections"),
        ((q, None, pos, (20, 20)), {}, "do not fit"),
        ((q, None, pos, (0, 0)), {}, "do not fit"),
        ((q, None, pos, (4, 4, 4)), {}, "positions must be"),
        ((q, None, pos.double(), (4, 4)), {}, "float32 or integers"),
        ((q, None, pos, (4, 4)), dict(pairing="quarter"), "pairing"),
        ((q, None, pos, (4, 4)), dict(spectrum="own"), "spectrum"),
        ((q, None, pos, (4, 4)), dict(base=0.0), "base"),
    ]:
        with pytest.raises(ValueError, match=text):
            rotary_axes(*args, **kw)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dim,pairs", [(8, 1), (9, 1), (11, 4), (17, 8), (18, 8), (20, 8), (24, 8), (25, 8), (45, 17),
                                       (64, 31), (70, 32), (31, 15), (16, 3), (22, 7)])
def test_pairs_and_rest_beside_the_vector(dim, pairs, pairing, dtype):
    """Pair counts and copied rests that fill no vector, one vector, or one and a part, out of a packed
    projection at an odd element."""
    rows, pos = data(53, 5, dim + 3, dtype, dim, 1)
    for x in (rows[:, :, :dim], rows[:, 1:, 3:]):
        got, other = rotary_axes(x, rows[:, :2, 1:dim + 1], pos, (pairs,), pairing=pairing)
        check(got, formula(x, pos, (pairs,), 10000.0, pairing, "axis"))
        check(other, formula(rows[:, :2, 1:dim + 1], pos, (pairs,), 10000.0, pairing, "axis"))
        assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])
