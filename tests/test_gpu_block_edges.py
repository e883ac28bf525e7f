"""What is not finite beside the block operators' dropped, masked and padded elements, and calls at their limits."""
import math

import pytest
import torch

import block_ref as R
from amdsplat import dropout, gated_scan, linear, norm, residual_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rand(seed, *shape, dtype=F32, gain=1.0):
    return (gain * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("width", [77, 96, 1100, 4104])
def test_a_dropped_elements_gradient_is_zero(width, post, bad):
    """Whatever arrives at it (h's gradient alone is spoiled, so no sum over a row is), as from `dropout` by itself."""
    rows, seed, p = 11, 7, 0.4
    x, y = rand(1, rows, width).requires_grad_(True), rand(2, rows, width, dtype=BF16).requires_grad_(True)
    w, gate, pw = rand(3, width), rand(4, width), rand(5, width).requires_grad_(True) if post else None
    d_h, d_n = rand(6, rows, width), rand(7, rows, width, dtype=BF16)
    dropped = R.keep(rows, width, seed, 0, p).to(DEV) == 0
    leaves = [y] + ([pw] if post else [])

    def grads(d_h, gate):
        h, n = residual_norm(x, y, w, post_weight=pw, gate=gate, dropout=p, seed=seed)
        return torch.autograd.grad((h, n), leaves, (d_h, d_n))

    want = grads(d_h, gate)
    got = grads(torch.where(dropped, torch.full_like(d_h, bad), d_h), gate)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert bool((want[0][dropped] == 0).all()) or post


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [7, 70])
def test_relus_gradient_beside_what_is_not_finite(rows, dtype):
    """With the identity for a weight the products are exact: z is x, and x's gradient the output's where z is positive, 0 where it is
    not, whatever arrives there. A row of NaN lets its gradient through, as torch's relu does."""
    n = 64
    x = rand(1, rows, n, dtype=dtype)
    bias = torch.zeros(n, device=DEV, requires_grad=True)
    eye, d = torch.eye(n, dtype=dtype, device=DEV), rand(2, rows, n, dtype=dtype)
    d = torch.where((x <= 0) & (rand(3, rows, n) > 0), torch.full_like(d, math.inf), d)
    x[5, 3] = math.nan  # (all of z's row 5: 0 times NaN)
    d[5] = rand(4, n, dtype=dtype)
    want = torch.where(x <= 0, torch.zeros_like(d), d)
    want[5] = d[5]
    for b in (None, bias):
        leaves = [x.clone().requires_grad_(True)] + ([] if b is None else [b])
        got = torch.autograd.grad(linear(leaves[0], eye, b, activation="relu"), leaves, d)
        assert torch.equal(got[0], want)
        if b is not None:
            size = want.double().abs().sum(0)
            assert bool(((got[1].double() - want.double().sum(0)).abs() <= (rows + 2) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 9, 40, 300])
def test_gradients_of_rows_that_overlap(rows, dtype):
    """Windows that move by a quarter of their width (or a single row of stride 0), with an infinity in the last one: in the
    gradients it reaches its own columns, as in those of copies."""
    k, step = 128, 32 if rows > 1 else 0
    flat = rand(1, (rows - 1) * step + k, dtype=dtype)
    flat[(rows - 1) * step + 40] = math.inf
    windows, plain, d = flat.as_strided((rows, k), (step, 1)), rand(2, 40, k, dtype=dtype), rand(3, rows, 40, dtype=dtype)

    def grads(x, w, d, bias=None):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        return torch.autograd.grad(linear(x, w, bias), (x, w), d)

    for a, b in ((windows, plain), (plain, windows)):
        g = d if a is windows else d.t().contiguous()
        got, want = grads(a, b, g), grads(a.clone(memory_format=torch.contiguous_format), b.clone(memory_format=torch.contiguous_format), g)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        finite = torch.ones(k, dtype=torch.bool, device=DEV)
        finite[[i for i in range(k) if not math.isfinite(float(windows[:, i].float().abs().max()))]] = False
        assert 0 < int((~finite).sum()) <= 3
        assert bool(torch.isfinite(got[1] if a is windows else got[0])[:, finite].all())


@pytest.mark.parametrize("width", [50, 64, 2000, 5000])
def test_a_norm_that_goes_nowhere_adds_nothing(width):
    """h alone is used, and rows of it are not finite: x's gradient is h's, the next norm's weight has none."""
    x, y, w = rand(1, 9, width), rand(2, 9, width).requires_grad_(True), rand(3, width).requires_grad_(True)
    x[2, 5], x[4, 49], x[6, 0] = math.inf, math.nan, -math.inf
    x.requires_grad_(True)
    gate, d = rand(4, width), rand(5, 9, width)
    for kind in ("rms", "layer"):
        h, _ = residual_norm(x, y, w, w, kind=kind, gate=gate, scale=0.5)
        dx, dy, dw = torch.autograd.grad(h, (x, y, w), d)
        assert torch.equal(dx, d) and bool((dw == 0).all())
        want = (0.5 * gate.double() * d.double())
        assert bool(((dy.double() - want).abs() <= 2 * 2.0 ** -24 * want.abs()).all())


def test_rows_of_several_launches():
    """2^26 rows and more: norms of heads over a long batch. Pieces of the rows give the same bits; the dropout's rows go on being
    counted, so the parts of a branch by themselves give h and n."""
    t, c, piece = (1 << 26) + 5, 8, 1 << 23
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(t, c, generator=g, device=DEV, dtype=BF16).requires_grad_(True)
    w = rand(2, c).requires_grad_(True)
    n = norm(x, w)
    with torch.no_grad():
        for at in range(0, t, piece):
            assert torch.equal(n[at:at + piece], norm(x[at:at + piece], w)), at
    d = torch.randn(t, c, generator=g, device=DEV, dtype=BF16)
    dx, dw = torch.autograd.grad(n, (x, w), d)
    want, size = torch.zeros(2, c, dtype=torch.float64, device=DEV)
    for at in range(0, t, piece):
        r = slice(at, at + piece)
        near = x[r].detach().requires_grad_(True)
        assert torch.equal(dx[r], torch.autograd.grad(norm(near, w), near, d[r])[0])
        hat = x[r].detach().double()
        hat *= (hat.square().mean(1, keepdim=True) + 1e-6).rsqrt()
        want += (d[r].double() * hat).sum(0)
        size += (d[r].double() * hat).abs().sum(0)
    # 512 workgroups of four rows at a time, their sums and their join
    assert bool(((dw.double() - want).abs() <= (t / 2048 + 600 + 32) * 2.0 ** -24 * size).all())
    del n, d, dx
    x = x.detach()
    y = torch.randn(t, c, generator=g, device=DEV, dtype=BF16)
    h, n = residual_norm(x.float(), y, w.detach(), dropout=0.25, seed=9)
    for at in range(0, t, piece):
        r = slice(at, at + piece)
        assert torch.equal(n[r], norm(h[r], w.detach(), dtype=BF16)), at
    kept = h != x.float()
    assert torch.equal(kept, (dropout(torch.ones_like(y), 0.25, 9) != 0) & (y != 0) & kept)
    missed = (dropout(torch.ones_like(y), 0.25, 9) != 0) & ~kept  # only where the branch vanishes beside the stream
    assert bool((y[missed].float().abs() <= 2.0 ** -23 * x[missed].float().abs()).all())


@pytest.mark.parametrize("dtype,shape", [
    (BF16, (2763, 3821, 4951)), (BF16, (3099, 4101, 201)), (BF16, (981, 1113, 3081)), (BF16, (10009, 1167, 307)), (BF16, (2305, 1565, 1801)),
    (F32, (943, 1099, 2491)), (F32, (1299, 3493, 1027)), (F32, (8251, 835, 59))])
def test_a_projection_is_the_same_with_and_without_gradients(dtype, shape):
    """What is kept for the backward pass changes neither where the contraction is cut nor a bit of the result."""
    m, n, k = shape
    x, w, b = rand(1, m, k, dtype=dtype), rand(2, n, k, dtype=dtype, gain=1 / math.sqrt(k)).requires_grad_(True), rand(3, n)
    for bias in (None, b):
        out = linear(x, w, bias, activation="gelu")
        assert out.requires_grad
        with torch.no_grad():
            assert torch.equal(out.detach(), linear(x, w, bias, activation="gelu"))


def test_a_recurrence_without_tokens():
    """Every document is empty: states go through, and so do their gradients."""
    for docs in (1, 5, 70, 300):
        x = torch.zeros(0, 20, device=DEV, requires_grad=True)
        initial = rand(1, docs, 20).requires_grad_(True)
        offsets = None if docs == 1 else torch.zeros(docs + 1, dtype=torch.int32, device=DEV)
        for reverse in (False, True):
            y, state = gated_scan(x, x, x, offsets=offsets, initial=initial, reverse=reverse, return_state=True)
            assert y.shape == (0, 20) and torch.equal(state, initial)
            d = rand(2, docs, 20)
            dx, di = torch.autograd.grad((y, state), (x, initial), (torch.zeros_like(y), d))
            assert dx.shape == (0, 20) and torch.equal(di, d)
            assert gated_scan(x, x, offsets=offsets, return_state=True)[1].eq(0).all()


@pytest.mark.parametrize("tokens", [3, 70])
def test_the_widest_recurrence(tokens):
    """2^20 channels; channels do not reach each other, so some of them alone give the same bits."""
    c = 1 << 20
    g = torch.Generator(device=DEV).manual_seed(1)
    x, f, o, d = (torch.randn(tokens, c, generator=g, device=DEV, dtype=BF16) for _ in range(4))
    offsets = torch.tensor([0, 1, tokens], dtype=torch.int32, device=DEV)
    parts = (slice(0, 8), slice(c // 2 - 4, c // 2 + 4), slice(c - 8, c))

    def run(x, f, o, d):
        v = [t.detach().clone().requires_grad_(True) for t in (x, f, o)]
        y, state = gated_scan(*v, offsets=offsets, return_state=True)
        return y.detach(), state.detach(), *torch.autograd.grad((y, state), v, (d, torch.ones_like(state)))

    whole = run(x, f, o, d)
    for p in parts:
        for a, b in zip(whole, run(x[:, p], f[:, p], o[:, p], d[:, p].contiguous())):
            assert torch.equal(a[:, p], b)
    with pytest.raises(ValueError, match="width"):
        gated_scan(*[torch.empty(1, c + 1, device=DEV, dtype=BF16)] * 2)


def test_dropout_over_the_longest_dimension():
    """2^31 - 1 elements in one row: the first ones are those of a shorter row, the last ones the generator's."""
    n = (1 << 31) - 1
    x = torch.ones(n, dtype=BF16, device=DEV)
    out = dropout(x, 0.25, 9)
    assert torch.equal(out[:1 << 20], dropout(x[:1 << 20], 0.25, 9))
    for group in (n // 8, n // 8 - 1, n // 16):
        words = R.philox([group, 0, 0, 0], [9, 0])
        bits = torch.tensor([h for word in words for h in (word & 0xffff, word >> 16)])
        mine = out[8 * group:8 * group + 8]
        assert torch.equal(mine == 0, (bits < 16384).to(DEV)[:len(mine)])
    kept = float((out != 0).sum()) / n
    assert abs(kept - 0.75) < 6 * math.sqrt(0.75 * 0.25 / n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_widest_projections(dtype):
    """2^19 inputs, 2^19 outputs, rows nearly 2^20 elements apart; few rows and tiles; all gradients, against float64."""
    from test_gpu_linear import check

    wide = 1 << 19
    g = torch.Generator(device=DEV).manual_seed(3)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    far = torch.zeros(40, (1 << 20) - 8, dtype=dtype, device=DEV)
    for rows in (9, 40):
        far[:rows, 8:wide + 8] = randn(rows, wide)
        check(far[:rows, 8:wide + 8], randn(24, wide) / 700, randn(24).float(), "silu")
        check(randn(rows, 64), randn(wide, 64) / 8, None, "none", randn(rows, wide).float())
    for shape in ((4, wide + 8), (wide + 8, 4)):
        with pytest.raises(ValueError, match="provided"):
            linear(torch.zeros(2, shape[1], dtype=dtype, device=DEV), torch.zeros(shape, dtype=dtype, device=DEV))


@pytest.mark.parametrize("rows,k", [(200, 101), (9, 101), (40, 128)])
def test_copied_rows_in_a_captured_step(rows, k):
    """What is copied first (rows of an odd length, windows that overlap) is copied again in every replay."""
    flat = rand(1, rows * 160, dtype=BF16)
    x = flat.as_strided((rows, k), (32, 1) if k == 128 else (k, 1)).detach().requires_grad_(True)
    w, b = rand(2, 72, k, dtype=BF16).requires_grad_(True), rand(3, 72).requires_grad_(True)
    d = rand(4, rows, 72, dtype=BF16)

    def step():
        out = linear(x, w, b, activation="gelu")
        first = torch.autograd.grad(out, (x, w, b), d, retain_graph=True)
        second = torch.autograd.grad(out, (x, w, b), d)
        return out.detach(), *first, *second

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        flat.copy_(rand(seed, rows * 160, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got[1:4], got[4:]))
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_two_threads():
    """Calls from two threads on streams of their own, refused ones among them: results and messages are each call's own."""
    from concurrent.futures import ThreadPoolExecutor

    x, w = rand(1, 300, 200, dtype=BF16), rand(2, 136, 200, dtype=BF16)
    y, s = rand(3, 500, 640), rand(4, 640)
    want = linear(x, w, activation="gelu"), norm(y, s), gated_scan(y, y)
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(30):
                got = linear(x, w, activation="gelu"), norm(y, s), gated_scan(y, y)
                with pytest.raises(Exception, match="eps" if i else "activation"):
                    norm(y, s, eps=-1.0) if i else linear(x, w, activation="x")
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        return True

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(work, range(2)))
