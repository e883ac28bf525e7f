"""The recurrence over sequences whose parts take several steps (above 65536 tokens), with memories as long as the sequence, so that
states and their gradients go from step to step and from part to part. The reference is float64 by doubling: after step k every
row holds the product and the sum of the 2^k rows up to it. Bounds are those of test_gpu_scan.py: forget gates of 9 to 15
have 15 half-steps of the exponential's argument, where its 12 have 12, and its 2^-15 of the size is 512 of them."""
import math

import pytest
import torch

from amdsplat import _lib, gated_scan
from test_gpu_scan import near

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rand(seed, *shape, dtype=F32, gain=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (gain * torch.randn(shape, generator=g, device=DEV) + shift).to(dtype)


def recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t along the first axis from h = 0."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat((b[:step], b[step:] + a[step:] * b[:-step]))
        a = torch.cat((a[:step], a[step:] * a[:-step]))
        step *= 2
    return b


def reference(x, f, o, cuts, initial, reverse, d_y, d_state):
    """(values, sizes), documents cuts[d] .. cuts[d + 1] that cover all tokens."""
    turn = (lambda v: v.flip(0)) if reverse else (lambda v: v)
    x, f, o, initial, d_y, d_state = (turn(t.detach().double()) for t in (x, f, o, initial, d_y, d_state))
    lens = torch.tensor([b - a for a, b in zip(cuts, cuts[1:])], device=DEV)
    lens = turn(lens)
    some, ends = lens > 0, lens.cumsum(0)
    first, last = (ends - lens)[some], ends[some] - 1
    a, rest, p = torch.sigmoid(f), torch.sigmoid(-f), torch.sigmoid(o)
    inner = a.clone()
    inner[first] = 0
    later = torch.cat((inner[1:], torch.zeros_like(inner[:1])))
    value, size = {}, {}
    for to, sign in ((value, lambda v: v), (size, torch.abs)):  # the sizes: every term's absolute value
        b = rest * sign(x)
        b[first] += a[first] * sign(initial)[some]
        h = recurrence(inner, b)
        state = sign(initial).clone()
        state[some] = h[last]
        d = sign(d_y * o * p)
        d[last] += sign(d_state)[some]
        d = recurrence(later.flip(0), d.flip(0)).flip(0)
        before = torch.cat((torch.zeros_like(h[:1]), h[:-1]))
        before[first] = sign(initial)[some]
        d_initial = sign(d_state).clone()
        d_initial[some] = a[first] * d[first]
        reach = before - x if to is value else before + x.abs()
        to.update(y=turn(h * sign(o * p)), state=turn(state), d_x=turn(d * rest), d_forget=turn(d * reach * a * rest),
                  d_gate=turn(sign(d_y) * h * (p + sign(o) * p * (1 - p))), d_initial=turn(d_initial))
    return value, size


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("tokens,width,dtype,cuts", [
    (150001, 4, F32, [0, 150001]),
    (150001, 5, F32, [0, 0, 1, 131071, 131071, 149990, 150001]),
    (70003, 3, F32, [0, 70003]),
    (70003, 260, F32, [0, 300, 70003]),
    (140000, 8, BF16, [0, 139999, 140000, 140000]),
])
def test_parts_of_several_steps(tokens, width, dtype, cuts, reverse):
    chunks = _lib.size_call("gs_gated_scan_chunks", tokens)
    # the workspace: a chunk's map is 8 bytes a channel, a part's with its state 12
    rest = _lib.size_call("gs_gated_scan_workspace_size", tokens, width) - (chunks * width * 8 + 15) // 16 * 16
    parts = rest // (12 * width)
    assert 1 < parts and chunks > 8 * parts  # eight chunks are a step
    docs = len(cuts) - 1
    x, o = rand(1, tokens, width, dtype=dtype, shift=0.5), rand(3, tokens, width, dtype=dtype)
    f = rand(2, tokens, width, shift=12.0).clamp(9, 15).to(dtype)
    initial = rand(4, docs, width, gain=3.0)
    d_y, d_state = rand(5, tokens, width, dtype=dtype), rand(6, docs, width, gain=100.0)
    leaves = [t.requires_grad_(True) for t in (x, f, o, initial)]
    table = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    y, state = gated_scan(x, f, o, offsets=table, initial=initial, reverse=reverse, return_state=True)
    grads = torch.autograd.grad((y, state), leaves, (d_y, d_state))
    value, size = reference(x, f, o, cuts, initial, reverse, d_y, d_state)
    near(y, value["y"], size["y"], "y")
    near(state, value["state"], size["state"], "state")
    for name, g in zip(("d_x", "d_forget", "d_gate", "d_initial"), grads):
        near(g, value[name], size[name], name)
    # what went in at one end of the longest document is there at the other
    longest = max(range(docs), key=lambda d: cuts[d + 1] - cuts[d])
    with torch.no_grad():
        moved = initial.clone()
        moved[longest] += 1.0
        _, other = gated_scan(x, f, o, offsets=table, initial=moved, reverse=reverse, return_state=True)
    share = torch.sigmoid(f[cuts[longest]:cuts[longest + 1]].detach().double()).log().sum(0).exp()
    assert float(share.max()) > 0.1
    room = 2.0 ** -14 * (size["state"][longest] + 1)
    assert bool(((other - state)[longest].double() - share).abs().le(room).all())
    assert math.isfinite(float(share.sum()))
