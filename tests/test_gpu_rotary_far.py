"""amdsplat.rotary_axes at far positions, against the formula in extended precision.

Bound: as near zero (test_gpu_rotary.py), for the angle is reduced to a turn before it is rounded to float32. In
64 bits n turns are known to n 2^-52 of a turn, 2 pi n 2^-52 in the angle: added below, it reaches the 2^-22 of the
rest at 2^27 turns."""
import numpy as np
import pytest
import torch

from amdsplat import rotary_axes

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("reach", [24, 27, 29, 30, 31, 33])
def test_far_positions(reach, pairing):
    tokens, pairs = 200, 32
    g = torch.Generator().manual_seed(reach)
    x = torch.randn(tokens, 2, 64, generator=g)
    # whole positions that float32 holds, over the whole reach and of both signs
    pos = torch.randint(-(1 << 24), 1 << 24, (tokens, 1), generator=g).float() * 2.0 ** (reach - 24)
    got = rotary_axes(x.to(DEV), None, pos.to(DEV), (pairs,), pairing=pairing).cpu().double()
    freq = np.longdouble(10000.0) ** -(np.arange(pairs, dtype=np.longdouble) / pairs)
    turns = pos.numpy().astype(np.longdouble) * freq / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    part = 2 * np.longdouble("3.14159265358979323846264338327950288") * (turns - np.rint(turns))
    c, s = (torch.from_numpy(f(part).astype(np.float64))[:, None] for f in (np.cos, np.sin))
    a, b = (slice(0, pairs), slice(pairs, 2 * pairs)) if pairing == "half" else (slice(0, 64, 2), slice(1, 64, 2))
    u, w = x[..., a].double(), x[..., b].double()
    near = 2.0 ** -22 + 2 * np.pi * 2.0 ** -52 * torch.from_numpy(np.abs(turns).astype(np.float64))[:, None]
    for value, mine in ((u * c - w * s, got[..., a]), (u * s + w * c, got[..., b])):
        off = (mine - value).abs()
        bound = near * (u.abs() + w.abs()) + 2.0 ** -24 * value.abs()
        assert bool((off <= bound).all()), float((off / bound).max())
