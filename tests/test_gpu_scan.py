"""GPU parity of amdsplat.gated_scan against the recurrence in float64, token by token.

Bound: the smaller of a and 1 - a is off by a few float32 roundings and |f| 2^-23 of itself (the exponential's argument),
32 steps of 2^-24 for |f| <= 12. A step's share of that is (1 - a) or a times a difference of what the recurrence of
absolute values (the size) holds, and a steady recurrence divides the sum of the shares by 1 - a, so the state is off by at most
2 * 32 steps of its size, by 2 * 16 for the roundings of a chunk's sixteen steps, and by another 32 for the maps of
chunks: 2^-17. An output gate adds its own 2^-18, gradients multiply two such values: 2^-15 of the size covers both. Then one
rounding to the type."""
import math

import pytest
import torch

import block_ref as R
from amdsplat import gated_scan

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DT = [torch.bfloat16, torch.float32]


def near(got, value, size, what):
    off = (got.detach().double().cpu() - value.cpu()).abs()
    bound = 2.0 ** -15 * size.cpu() + UNIT[got.dtype] * value.cpu().abs() + 1e-37
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float((off / bound).max()))


def data(seed, tokens, width, dtype, shift=2.0):
    g = torch.Generator().manual_seed(seed)
    x, f, o = (torch.randn(tokens, width, generator=g) for _ in range(3))
    return [t.to(dtype).to(DEV) for t in (x, (1.5 * f + shift).clamp(-12, 12), o)]


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def check(x, f, o=None, offsets=None, initial=None, reverse=False, through="both"):
    leaves = {n: t.detach().requires_grad_(True) for n, t in (("x", x), ("forget", f), ("gate", o), ("initial", initial))
              if t is not None}
    table = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=DEV)
    docs = 1 if offsets is None else len(offsets) - 1
    y, state = gated_scan(**leaves, offsets=table, reverse=reverse, return_state=True)
    assert y.dtype == x.dtype and state.dtype == torch.float32 and state.shape == (docs, x.shape[1])
    d_y = rand(91, *x.shape, dtype=x.dtype) if through != "state" else None
    d_state = rand(92, docs, x.shape[1]) if through != "y" else None
    outs, ds = zip(*[(a, b) for a, b in ((y, d_y), (state, d_state)) if b is not None])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ds)))
    cpu = {n: t.detach().cpu() for n, t in leaves.items()}
    value, size = R.gated_scan(**cpu, offsets=offsets, reverse=reverse, d_y=None if d_y is None else d_y.cpu(),
                               d_state=None if d_state is None else d_state.cpu())
    near(y, value["y"], size["y"], "y")
    near(state, value["state"], size["state"], "state")
    for n, g in grads.items():
        near(g, value["d_" + n], size["d_" + n], "d_" + n)
    with torch.no_grad():
        y2, s2 = gated_scan(**leaves, offsets=table, reverse=reverse, return_state=True)
    assert torch.equal(y, y2) and torch.equal(state, s2)
    assert torch.equal(y, gated_scan(**leaves, offsets=table, reverse=reverse))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 129, 300])
def test_lengths(tokens, gated, reverse, dtype):
    x, f, o = data(tokens, tokens, 20, dtype)
    check(x, f, o if gated else None, initial=rand(5, 1, 20) if tokens % 2 else None, reverse=reverse)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("width", [1, 3, 4, 5, 64, 255, 256, 257, 520])
def test_widths(width, dtype):
    x, f, o = data(width, 70, width, dtype)
    check(x, f, o, offsets=[0, 30, 70], initial=rand(5, 2, width))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("offsets", [
    [0, 0], [0, 200], [3, 190], [0, 0, 0, 200, 200], [0, 1, 2, 3, 200], [0, 16, 32, 200], [0, 15, 17, 33, 200, 200],
    [7, 7, 8, 8, 150, 150], list(range(0, 201)), [0] * 70 + [100] * 70 + [200], [200, 200], [0, 199, 200]])
def test_documents(offsets, reverse, dtype):
    x, f, o = data(len(offsets), 200, 12, dtype)
    check(x, f, o, offsets=offsets, initial=rand(5, len(offsets) - 1, 12), reverse=reverse)
    check(x, f, None, offsets=offsets, reverse=reverse, through="y")
    check(x, f, o, offsets=offsets, reverse=reverse, through="state")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("tokens,offsets", [
    (30, [0, 5, 20, 30]), (31, [2, 2, 18, 25]), (32, [0, 0, 32, 32]), (17, [16, 17]), (20, [3] * 40 + [19]), (9, [0, 9] + [9] * 1030),
    (200, [5] * 50 + [9] * 60 + [120] * 40 + [190] * 60), (200, [0] * 100 + [200] * 101), (200, [200] * 201),
    (250, list(range(0, 251)) + [250] * 6), (250, list(range(0, 251)) + [250] * 7), (70, [i // 2 for i in range(8, 141)])])
def test_documents_of_few_tokens(tokens, offsets, reverse, dtype):
    """No more tokens than 32, or than documents: a wavefront walks a document's."""
    x, f, o = data(len(offsets), tokens, 20, dtype)
    check(x, f, o, offsets=offsets, initial=rand(5, len(offsets) - 1, 20), reverse=reverse)
    check(x, f, None, offsets=offsets, reverse=reverse, through="state")


@pytest.mark.parametrize("reverse", [False, True])
def test_many_parts(reverse):
    """More chunks than one part has, and parts of more than one step, in one document and in many."""
    x, f, o = data(3, 40000, 5, torch.float32)
    cuts = [0, 17, 5000, 5000, 20481, 39990]
    check(x, f, o, offsets=cuts, initial=rand(5, 5, 5), reverse=reverse)
    check(x, f, None, initial=rand(5, 1, 5), reverse=reverse)


def test_single_tokens_continue():
    """Tokens one at a time against the state, as they would have come together; many scenes at once."""
    docs, width = 70, 300
    x, f, o = data(6, 5 * docs, width, torch.bfloat16)
    x, f, o = (t.view(5, docs, width) for t in (x, f, o))
    at = torch.arange(docs + 1, dtype=torch.int32, device=DEV)
    state, ys = None, []
    for t in range(5):
        y, state = gated_scan(x[t], f[t], o[t], offsets=at, initial=state, return_state=True)
        ys.append(y)
    together = [t.transpose(0, 1).reshape(-1, width) for t in (x, f, o)]
    y, last = gated_scan(*together, offsets=5 * at, return_state=True)
    # the same steps in the same order, but for the rounding of states between calls: none
    want, size = R.gated_scan(*[t.cpu() for t in together], offsets=(5 * at).tolist())
    near(torch.stack(ys, 1).reshape(-1, width), want["y"], size["y"], "y")
    near(y, want["y"], size["y"], "y")
    near(state, want["state"], size["state"], "state")
    near(last, want["state"], size["state"], "state")


def test_strides():
    rows = rand(1, 90, 3 * 33 + 2)
    for dtype in DT:
        r = rows.to(dtype)
        for x, f, o in ((r[:, :33], r[:, 33:66], r[:, 66:99]), (r[:, 1:34], r[:, 35:68], r[:, 68:]),
                        (r[::2, :33], r[::2, 40:73], None), (r[:1, :33].expand(90, 33), r[:, 33:66], r[:, :33].t().contiguous().t())):
            check(x, f, o)


def test_far_memories_and_closed_gates():
    """Gates from fully closed to a memory of 2^17 tokens: the state's bound holds relative to its size. f up to 20 raises the
    exponential's share of the bound from 12 to 20 of 2^-23, which 2^-15 covers."""
    for shift in (-30.0, -8.0, 8.0, 12.0, 20.0):
        x = rand(1, 5000, 8) + 1
        f = torch.full((5000, 8), shift, device=DEV)
        y, state = gated_scan(x, f, initial=torch.full((1, 8), 1e4, device=DEV), return_state=True)
        value, size = R.gated_scan(x.cpu(), f.cpu(), initial=torch.full((1, 8), 1e4))
        near(y, value["y"], size["y"], shift)
        near(state, value["state"], size["state"], shift)
    f = torch.tensor([math.inf, -math.inf], device=DEV).repeat(40, 4)
    x = rand(2, 40, 8)
    y = gated_scan(x, f, initial=torch.full((1, 8), 3.0, device=DEV))
    assert y[:, ::2].eq(3.0).all() and torch.equal(y[:, 1::2], x[:, 1::2])


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_documents_do_not_reach_each_other(bad, reverse):
    x, f, o = data(7, 400, 8, torch.float32)
    cuts = [0, 20, 130, 131, 290, 400]
    table = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    d = rand(8, 400, 8)

    def run(x, f, o, d):
        x, f, o = (t.detach().requires_grad_(True) for t in (x, f, o))
        y, s = gated_scan(x, f, o, offsets=table, reverse=reverse, return_state=True)
        return (y, s, *torch.autograd.grad((y, s), (x, f, o), (d, torch.ones_like(s))))

    want = run(x, f, o, d)
    for spoiled in range(4):
        v = [x.clone(), f.clone(), o.clone(), d.clone()]
        v[spoiled][20:130:7] = bad
        v[spoiled][290:400:3] = bad
        for i, (a, b) in enumerate(zip(run(*v), want)):
            keep = [0, 2, 3] if i == 1 else [*range(0, 20), *range(130, 290)]
            assert torch.equal(a[keep], b[keep]), (spoiled, i)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_documents_of_few_tokens_do_not_reach_each_other(bad, reverse):
    """As above where a wavefront walks a document, tokens of none among them; then offsets outside the tensor, and a
    replayed graph whose documents move between replays."""
    tokens, cuts = 200, [5] * 50 + [9] * 60 + [120] * 40 + [131] * 30 + [190] * 30
    x, f, o = data(17, tokens, 12, torch.float32)
    table = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    docs, d = len(cuts) - 1, rand(18, tokens, 12)
    initial = rand(19, docs, 12)

    def run(x, f, o, d, table=table):
        x, f, o, i = (t.detach().requires_grad_(True) for t in (x, f, o, initial))
        y, s = gated_scan(x, f, o, offsets=table, initial=i, reverse=reverse, return_state=True)
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), (x, f, o, i), (d, torch.ones_like(s))))

    want = run(x, f, o, d)
    assert all(bool((want[i][:5] == 0).all()) and bool((want[i][190:] == 0).all()) for i in (0, 2, 3, 4))
    others = [i for i in range(docs) if i != cuts.index(120) - 1]
    for spoiled in range(4):
        v = [x.clone(), f.clone(), o.clone(), d.clone()]
        v[spoiled][9:120:7] = bad
        v[spoiled][:5] = bad
        v[spoiled][190:] = bad
        for i, (a, b) in enumerate(zip(run(*v), want)):
            keep = others if i in (1, 5) else [*range(0, 9), *range(120, tokens)]
            assert torch.equal(a[keep], b[keep]), (spoiled, i)
    outside = table.clone()
    outside[outside == 5], outside[outside == 190] = -7, 1 << 30
    inside = outside.clamp(0, tokens)
    assert all(torch.equal(a, b) for a, b in zip(run(x, f, o, d, outside), run(x, f, o, d, inside)))
    moving = table.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, f, o, d, moving)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, f, o, d, moving)
    for to in (table, inside, torch.arange(docs + 1, dtype=torch.int32, device=DEV).clamp(max=tokens), table):
        moving.copy_(to)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run(x, f, o, d, moving)))


def test_offsets_outside_the_tensor_are_cut():
    x, f, o = data(9, 100, 8, torch.float32)
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for got, want in (((-5, 40, 1000), (0, 40, 100)), ((0, 200, 300), (0, 100, 100))):
        a = gated_scan(x, f, o, offsets=t(*got), return_state=True)
        b = gated_scan(x, f, o, offsets=t(*want), return_state=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    # offsets that decrease: whatever comes, it stays in the tensors
    y, s = gated_scan(x, f, o, offsets=t(50, 20, 90, 10), return_state=True)
    assert y.shape == x.shape and s.shape == (3, 8)


def test_gradient_against_differences():
    """Linear in x and the initial state, so a difference of any step is the directional derivative: float32, with the
    two forwards' and the gradient's bounds."""
    x, f, o = data(10, 333, 24, torch.float32)
    way, w = rand(11, 333, 24), rand(12, 333, 24)
    x.requires_grad_(True)
    g, = torch.autograd.grad(gated_scan(x, f, o), x, w)
    with torch.no_grad():
        slope = float(((gated_scan(x + way, f, o).double() - gated_scan(x, f, o).double()) * w.double()).sum())
        mine = float((g.double() * way.double()).sum())
        sizes = [R.gated_scan(t.cpu(), f.cpu(), o.cpu())[1]["y"] for t in (x, x + way)]
        room = 2.0 ** -15 * float((sum(sizes) * w.double().abs().cpu()).sum()) * 2
    assert abs(mine - slope) <= room


def test_captured_with_its_backward():
    x, f, o = (t.requires_grad_(True) for t in data(13, 500, 64, torch.bfloat16))
    table = torch.tensor([0, 100, 500], dtype=torch.int32, device=DEV)
    d = rand(14, 500, 64, dtype=torch.bfloat16)

    def step():
        y = gated_scan(x, f, o, offsets=table)
        return y.detach(), *torch.autograd.grad(y, (x, f, o), d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for cut in (100, 1, 499, 250):
        table[1] = cut
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_on_a_side_stream():
    x, f, o = data(15, 700, 128, torch.bfloat16)
    want = gated_scan(x, f, o)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = gated_scan(x, f, o)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    x, t = z(10, 8), torch.tensor([0, 10], dtype=torch.int32, device=DEV)
    for args, kw, text in [
        ((z(10), z(10)), {}, "tokens, width"), ((x.half(), x.half()), {}, "float32 or bfloat16"), ((x, z(10, 7)), {}, "forget must"),
        ((x, x.bfloat16()), {}, "forget must"), ((x, x, z(9, 8)), {}, "gate must"), ((x, x.cpu()), {}, "forget must"),
        ((z(10, 0), z(10, 0)), {}, "width"), ((x, x), dict(offsets=t.long()), "offsets"), ((x, x), dict(offsets=t.cpu()), "offsets"),
        ((x, x), dict(offsets=t[:1]), "offsets"), ((x, x), dict(initial=z(2, 8)), "initial"),
        ((x, x), dict(initial=z(1, 8, dtype=torch.bfloat16)), "initial"), ((x.cpu(), x.cpu()), {}, "GPU"),
    ]:
        with pytest.raises(ValueError, match=text):
            gated_scan(*args, **kw)
