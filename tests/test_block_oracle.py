"""oracle/block_ref.py against differences and against torch's own gradients in float64, and dropout's generator against
its published test vectors."""
import pytest
import torch

import block_ref as R


def test_philox_vectors():
    """The known answers published with the generator (Random123's kat_vectors, philox4x32 with ten rounds)."""
    ones = [0xffffffff] * 4
    assert R.philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert R.philox(ones, ones[:2]) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert R.philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_factors_are_the_generators():
    seed, draw = 0x0123456789abcdef, 0x1f2e3d4c5b6a7988
    f = R.keep(3, 21, seed, draw, 0.3)
    t = round(0.3 * 65536)
    for row in range(3):
        for col in range(21):
            w = R.philox([col // 8, row, draw & 0xffffffff, draw >> 32], [seed & 0xffffffff, seed >> 32])[col % 8 // 2]
            bits = w >> 16 if col % 2 else w & 0xffff
            assert float(f[row, col]) == (0.0 if bits < t else 65536 / (65536 - t))
    assert R.keep(2, 8, 1, 0, 0.0).eq(1).all() and R.keep(400, 80, 1, 0, 0.5).count_nonzero() in range(15300, 16700)


def draws(seed, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g, dtype=torch.float64) for s in shapes]


def check_differences(f, tensors, grads, seed):
    """f: tensors -> scalar. The directional derivative by central differences, float64, step 1e-5: its error is
    some 1e-10 of the function's size."""
    for i, (t, grad) in enumerate(zip(tensors, grads)):
        way, = draws(seed + i, t.shape)
        at = lambda e: f(*[x + e * way if j == i else x for j, x in enumerate(tensors)])  # noqa: E731
        slope = float((at(1e-5) - at(-1e-5)) / 2e-5)
        mine = float((grad * way).sum())
        assert abs(slope - mine) <= 1e-6 * (1 + abs(mine)), (i, slope, mine)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "column", "token"])
def test_residual_norm(kind, post, gate):
    x, y, w, b, pw, pb, d_h, d_n = draws(1, (5, 12), (5, 12), (12,), (12,), (12,), (12,), (5, 12), (5, 12))
    g = {None: None, "column": draws(2, (12,))[0], "token": draws(2, (5, 12))[0]}[gate]
    k = R.keep(5, 12, 77, 3, 0.25)
    if not post:
        pw = pb = None
    given = {n: t for n, t in (("x", x), ("y", y), ("weight", w), ("bias", b), ("post_weight", pw), ("post_bias", pb),
                               ("gate", g)) if t is not None}

    def total(*ts):
        r, _ = R.residual_norm(**dict(zip(given, ts)), kind=kind, scale=0.7, factors=k)
        return (r["h"] * d_h).sum() + (r["n"] * d_n).sum()

    r, size = R.residual_norm(**given, kind=kind, scale=0.7, factors=k, d_h=d_h, d_n=d_n)
    check_differences(total, list(given.values()), [r["d_" + n] for n in given], 10)
    for name in r:
        assert bool((r[name].abs() <= size[name] * (1 + 1e-12)).all()), name


def test_norm_alone():
    x, w, d_n = draws(3, (4, 9), (9,), (4, 9))
    r, _ = R.residual_norm(x, None, w, kind="rms", d_n=d_n)
    want = x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
    assert torch.allclose(r["n"], want, rtol=1e-13)
    check_differences(lambda a, b: (R.residual_norm(a, None, b, kind="rms")[0]["n"] * d_n).sum(), [x, w],
                      [r["d_x"], r["d_weight"]], 20)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_gated_scan(gated, reverse):
    x, f, o, h, d_y, d_s = draws(4, (11, 3), (11, 3), (11, 3), (4, 3), (11, 3), (4, 3))
    at = [1, 4, 4, 9, 10]
    given = dict(x=x, forget=f, **({"gate": o} if gated else {}), initial=h)

    def total(*ts):
        r, _ = R.gated_scan(**dict(zip(given, ts)), offsets=at, reverse=reverse)
        return (r["y"] * d_y).sum() + (r["state"] * d_s).sum()

    r, size = R.gated_scan(**given, offsets=at, reverse=reverse, d_y=d_y, d_state=d_s)
    check_differences(total, list(given.values()), [r["d_" + n] for n in given], 30)
    assert r["y"][[0, 10]].eq(0).all() and r["d_x"][[0, 10]].eq(0).all()
    assert r["state"][1].equal(h[1]) and r["d_initial"][1].equal(d_s[1])
    for name in r:
        assert bool((r[name].abs() <= size[name] * (1 + 1e-12)).all()), name


@pytest.mark.parametrize("how", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_linear(how):
    x, w, b, res, d = draws(5, (6, 7), (5, 7), (5,), (6, 5), (6, 5))
    r, size = R.linear(x, w, b, how, res, d)
    check_differences(lambda *t: (R.linear(t[0], t[1], t[2], how, res)[0]["out"] * d).sum(), [x, w, b],
                      [r["d_x"], r["d_weight"], r["d_bias"]], 40)
    f = torch.nn.functional
    z = x @ w.t() + b
    want = {"none": z, "relu": f.relu(z), "gelu": f.gelu(z), "gelu_tanh": f.gelu(z, approximate="tanh"), "silu": f.silu(z)}
    assert torch.allclose(r["out"], want[how] + res, rtol=1e-12, atol=1e-13)
    for name in r:
        assert bool((r[name].abs() <= size[name] * (1 + 1e-12)).all()), name
