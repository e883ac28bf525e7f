"""GPU parity of amdsplat.attention against the float64 oracle (oracle/attention_ref.py, which also
gives the elementwise bounds), at the sizes and masks where such kernels go wrong."""
import itertools

import pytest
import torch

import attention_ref as A
from amdsplat import attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check(got, want):
    for name, x in got.items():
        value, bound = want[name]
        x = x.detach().cpu().double()
        assert x.shape == value.shape, name
        fine = torch.isfinite(value)
        assert torch.equal(torch.isfinite(x), fine), (name, "finite in other places")
        assert torch.equal(x[~fine], value[~fine]), name
        off = (x - value).abs()[fine]
        over = off > bound[fine]
        assert not bool(over.any()), (name, int(over.sum()), float((off / bound[fine]).max()), float(off.max()))


def inputs(tq, tk, heads, kv_heads, dim, dtype, seed, gain=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (gain * torch.randn(tq, heads, dim, generator=g)).to(dtype)
    k, v = (torch.randn(tk, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.randn(tq, heads, dim, generator=g).to(dtype)


def run(q, k, v, d_out, **kw):
    q, k, v = (t.to(DEV).requires_grad_(d_out is not None) for t in (q, k, v))
    out, lse = attention(q, k, v, return_lse=True, **kw)
    r = {"out": out, "lse": lse}
    if d_out is not None:
        r["d_q"], r["d_k"], r["d_v"] = torch.autograd.grad(out, (q, k, v), d_out.to(DEV))
    return r


def both(lens, heads, kv_heads, dim, dtype, causal=False, prefix=None, softcap=0.0, seed=0, gain=1.5):
    at = offsets(lens)
    q, k, v, g = inputs(at[-1], at[-1], heads, kv_heads, dim, dtype, seed, gain)
    got = run(q, k, v, g, offsets=ints(at), causal=causal, prefix=None if prefix is None else ints(prefix),
              softcap=softcap)
    check(got, A.attention(q, k, v, at, at, causal=causal, prefix=prefix, softcap=softcap, d_out=g))


DT = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("mask", ["full", "causal", "prefix"])
def test_packed_documents(dim, mask, dtype):
    # lengths around the tiles' edges (32, 64, 128), one token, none
    lens = [1, 63, 0, 64, 65, 129, 31, 200]
    prefix = [0, 20, 0, 64, 1, 70, 99, 0] if mask == "prefix" else None
    both(lens, 4, 2, dim, dtype, mask != "full", prefix, seed=dim)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (16, 2), (5, 5), (7, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_head_groups(heads, kv_heads, causal, dtype):
    both([77, 130], heads, kv_heads, 64, dtype, causal, seed=heads)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("softcap,gain", [(30.0, 1.5), (5.0, 4.0), (50.0, 20.0), (200.0, 1.5)])
def test_capped_scores(softcap, gain, dim, dtype):
    both([97, 150], 4, 2, dim, dtype, True, [30, 0], softcap, seed=3, gain=gain)


@pytest.mark.parametrize("dtype", DT)
def test_large_scores(dtype):
    # scores of several hundred: the running maximum has to move, far keys underflow to nothing
    both([300, 513], 2, 2, 64, dtype, False, gain=40.0, seed=9)
    both([300, 513], 2, 1, 128, dtype, True, gain=40.0, seed=10)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 1), (128, 4, 1)])
def test_longer(dim, heads, kv_heads, dtype):
    both([1111], heads, kv_heads, dim, dtype, True, [200], 0.0, seed=4)
    both([2049], heads, kv_heads, dim, dtype, False, None, 0.0, seed=5)


@pytest.mark.parametrize("n", [1, 2, 3, 5, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
def test_one_document_of_each_length(n):
    both([n], 2, 1, 64, torch.bfloat16, True, seed=n)
    both([n], 2, 2, 32, torch.float32, False, seed=n)


def test_many_documents():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 9, (700,), generator=g).tolist()
    both(lens, 2, 1, 64, torch.bfloat16, True, seed=6)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("nq,causal", [(1, False), (1, True), (3, True), (40, True), (40, False)])
def test_cached_keys(nq, causal, dim, dtype):
    # caches of one capacity, filled to different lengths (none, fewer than the queries, all)
    cap, filled = 700, [700, 1, 0, 333, 64, nq, 650]
    heads, kv_heads, docs = 8, 2, len(filled)
    q, k, v, g = inputs(docs * nq, docs * cap, heads, kv_heads, dim, dtype, 11)
    q_at, k_at = offsets([nq] * docs), offsets([cap] * docs)
    want = A.attention(q, k, v, q_at, k_at, filled, causal=causal, d_out=g)
    for i, n in enumerate(filled):  # whatever the rest of the cache holds
        k[k_at[i] + n:k_at[i + 1]] = float("nan")
        v[k_at[i] + n:k_at[i + 1]] = float("inf") if i % 2 else float("nan")
    tables = dict(offsets=ints(q_at), k_offsets=ints(k_at), k_lengths=ints(filled), causal=causal)
    check(run(q, k, v, None, **tables), want)
    check(run(q, k, v, g, **tables), want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 1, 128), (32, 8, 128), (40, 1, 64)])
@pytest.mark.parametrize("keys", [1, 40, 1023, 9000])
def test_single_tokens(keys, heads, kv_heads, dim, dtype):
    q, k, v, _ = inputs(1, keys, heads, kv_heads, dim, dtype, keys)
    check(run(q, k, v, None), A.attention(q, k, v, [0, 1], [0, keys]))
    check(run(q, k, v, None, softcap=20.0, causal=True),
          A.attention(q, k, v, [0, 1], [0, keys], causal=True, softcap=20.0))


@pytest.mark.parametrize("dtype", DT)
def test_few_queries_over_ragged_caches(dtype):
    lens_q, lens_k = [1, 2, 0, 5, 1], [3000, 17, 900, 0, 4097]
    q_at, k_at = offsets(lens_q), offsets(lens_k)
    q, k, v, g = inputs(q_at[-1], k_at[-1], 6, 3, 64, dtype, 21)
    for causal in (False, True):
        got = run(q, k, v, g, offsets=ints(q_at), k_offsets=ints(k_at), causal=causal)
        check(got, A.attention(q, k, v, q_at, k_at, causal=causal, d_out=g))


@pytest.mark.parametrize("dtype", DT)
def test_rows_that_see_nothing(dtype):
    # fewer keys than queries: the first queries see none, or the prefix alone
    lens_q, lens_k = [100, 40, 70], [30, 0, 70]
    q_at, k_at = offsets(lens_q), offsets(lens_k)
    q, k, v, g = inputs(210, 100, 4, 2, 64, dtype, 22)
    for prefix in (None, [0, 5, 0], [12, 0, 80]):
        got = run(q, k, v, g, offsets=ints(q_at), k_offsets=ints(k_at), causal=True,
                  prefix=None if prefix is None else ints(prefix))
        check(got, A.attention(q, k, v, q_at, k_at, causal=True, prefix=prefix, d_out=g))


@pytest.mark.parametrize("dtype", DT)
def test_tokens_outside_the_documents(dtype):
    q, k, v, g = inputs(300, 300, 4, 2, 64, dtype, 23)
    at = [70, 200, 260]
    want = A.attention(q, k, v, at, at, d_out=g)
    for t in (k, v):
        t[:70] = t[260:] = float("nan")
    check(run(q, k, v, g, offsets=ints(at)), want)


def test_offsets_beyond_the_tensors_are_cut():
    q, k, v, g = inputs(100, 100, 2, 2, 64, torch.bfloat16, 24)
    want = A.attention(q, k, v, [0, 40, 100], [0, 40, 100], d_out=g)
    check(run(q, k, v, g, offsets=ints([-5, 40, 1 << 30])), want)
    check(run(q, k, v, g, offsets=ints([0, 40, 100]), k_lengths=ints([1 << 30, 60])), want)
    check(run(q, k, v, g, offsets=ints([0, 40, 100]), k_lengths=ints([-3, 60])),
          A.attention(q, k, v, [0, 40, 100], [0, 40, 100], [0, 60], d_out=g))


@pytest.mark.parametrize("dtype", DT)
def test_no_tokens(dtype):
    for tq, tk in ((0, 0), (0, 50), (50, 0)):
        q, k, v, g = inputs(tq, tk, 4, 2, 64, dtype, 25)
        at = ([0, tq], [0, tk])
        got = run(q, k, v, g, offsets=ints(at[0]), k_offsets=ints(at[1]))
        check(got, A.attention(q, k, v, *at, d_out=g))


@pytest.mark.parametrize("dtype", DT)
def test_strides_alignment_and_orders(dtype):
    tq, heads, kv, dim = 150, 4, 2, 40
    q, k, v, g = inputs(tq, tq, heads, kv, dim, dtype, 26)
    want = A.attention(q, k, v, [0, tq], [0, tq], causal=True, d_out=g)
    packed = torch.cat((q, k, v), 1).to(DEV)  # slices of one projection
    views = [packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]]
    by_head = [t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    by_dim = [t.to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (q, k, v)]
    shifted = []
    for t in (q, k, v):  # one element off 16-byte alignment
        buf = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)
        buf[1:] = t.flatten().to(DEV)
        shifted.append(buf[1:].view(t.shape))
    for a, b, c in (views, by_head, by_dim, shifted):
        a, b, c = (t.detach().requires_grad_(True) for t in (a, b, c))
        out, lse = attention(a, b, c, causal=True, return_lse=True)
        # the output's gradient in another order too
        d = g.to(DEV).permute(1, 2, 0).contiguous().permute(2, 0, 1)
        grads = torch.autograd.grad(out, (a, b, c), d)
        check(dict(out=out, lse=lse, d_q=grads[0], d_k=grads[1], d_v=grads[2]), want)
    # keys of one head for all (a broadcast input): its gradient is the heads' sum
    one_k, one_v = k[:, :1], v[:, :1]
    a, b, c = (t.to(DEV).requires_grad_(True) for t in (q, one_k, one_v))
    out = attention(a, b.expand(tq, heads, dim), c.expand(tq, heads, dim), causal=True)
    grads = torch.autograd.grad(out, (a, b, c), g.to(DEV))
    want = A.attention(q, one_k, one_v, [0, tq], [0, tq], causal=True, d_out=g)
    u = A.UNIT[dtype]
    full = A.attention(q, one_k.expand(tq, heads, dim), one_v.expand(tq, heads, dim), [0, tq], [0, tq], causal=True, d_out=g)
    check(dict(out=out, d_q=grads[0]), want)
    for x, name in ((grads[1], "d_k"), (grads[2], "d_v")):
        # each head's gradient was rounded, then torch summed them in the type
        bound = full[name][1].sum(1, keepdim=True) + 4 * u * full[name][0].abs().sum(1, keepdim=True)
        check({name: x}, {name: (want[name][0], bound)})


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [1, 3, 20, 50, 127])
def test_odd_head_sizes(dim, dtype):
    both([70, 33], 4, 2, dim, dtype, True, seed=dim)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(scale):
    q, k, v, g = inputs(90, 90, 2, 2, 64, torch.float32, 27)
    check(run(q, k, v, g, scale=scale), A.attention(q, k, v, [0, 90], [0, 90], scale=scale, d_out=g))


def test_same_bits_and_other_streams():
    at = offsets([500, 300, 900])
    q, k, v, g = (t.to(DEV) for t in inputs(at[-1], at[-1], 8, 2, 64, torch.bfloat16, 28))
    tables = dict(offsets=ints(at), causal=True)
    first = run(q, k, v, g, **tables)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            again = run(q, k, v, g, **tables)
        side.synchronize()
        for name, x in first.items():
            assert torch.equal(x, again[name]), name


def test_cache_past_32_bits():
    # 2.3e9 elements before the last document: its keys lie past 2^31 elements and 2^32 bytes
    tk, kv, dim, n = 2_250_000, 8, 128, 1000
    k = torch.empty(tk, kv, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(tk, kv, dim, dtype=torch.bfloat16, device=DEV)
    for nq, heads in ((1, 8), (150, 8)):
        q, kk, vv, _ = inputs(nq, n, heads, kv, dim, torch.bfloat16, 29)
        k[-n:], v[-n:] = kk.to(DEV), vv.to(DEV)
        out, lse = attention(q.to(DEV), k, v, offsets=ints([0, 0, nq]), k_offsets=ints([0, tk - n, tk]),
                             return_lse=True)
        check(dict(out=out, lse=lse), A.attention(q, kk, vv, [0, nq], [0, n]))


@pytest.mark.parametrize("softcap,causal", list(itertools.product([0.0, 10.0], [False, True])))
def test_gradients_against_differences(softcap, causal):
    """Directional derivatives of the float64 formula by central differences (step 1e-4: truncation
    1e-8 of third derivatives of order 1, rounding 1e-12)."""
    at = offsets([37, 70])
    q, k, v, g = inputs(at[-1], at[-1], 4, 2, 24, torch.float32, 30)
    got = run(q, k, v, g, offsets=ints(at), causal=causal, softcap=softcap)
    bounds = A.attention(q, k, v, at, at, causal=causal, softcap=softcap, d_out=g)
    gen = torch.Generator().manual_seed(31)

    def loss(q, k, v):
        total = 0.0
        for d in range(2):
            s = slice(at[d], at[d + 1])
            see = A.visible(at[d + 1] - at[d], at[d + 1] - at[d], causal, 0)
            for h in range(4):
                o = A.forward64(q[s, h], k[s, h // 2], v[s, h // 2], see, 24 ** -0.5, softcap)[0]
                total += float((o * g[s, h].double()).sum())
        return total

    x = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("d_q", "d_k", "d_v")):
        way = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-4 * way, x[i] - 1e-4 * way
        slope = (loss(*up) - loss(*down)) / 2e-4
        mine = float((got[name].cpu().double() * way).sum())
        tol = float((bounds[name][1] * way.abs()).sum()) + 1e-6 * float((bounds[name][0] * way).abs().sum())
        assert abs(mine - slope) <= tol, (name, mine, slope, tol)


def test_refusals():
    t = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    q, k = t(10, 4, 64), t(10, 2, 64)
    bad = [
        (dict(q=t(10, 64)), "tokens, heads"),
        (dict(q=t(10, 4, 64, dtype=torch.float16)), "dtype"),
        (dict(q=t(10, 4, 64, dtype=torch.float32)), "dtype"),
        (dict(q=torch.zeros(10, 4, 64, dtype=torch.bfloat16)), "GPU"),
        (dict(v=t(10, 2, 32)), "shape mismatch"),
        (dict(v=t(9, 2, 64)), "shape mismatch"),
        (dict(q=t(10, 4, 136), k=t(10, 2, 136), v=t(10, 2, 136)), "head size"),
        (dict(q=t(10, 3, 64)), "multiple"),
        (dict(k_offsets=ints([0, 10])), "without offsets"),
        (dict(offsets=ints([0])), "at least 2"),
        (dict(offsets=torch.tensor([0, 10], device=DEV)), "int32"),
        (dict(offsets=torch.tensor([0, 10], dtype=torch.int32)), "device"),
        (dict(offsets=ints([0, 10]), k_offsets=ints([0, 5, 10])), "entries"),
        (dict(q=t(7, 4, 64), offsets=ints([0, 7])), "pass k_offsets"),
        (dict(k_lengths=ints([1, 2])), "entries"),
        (dict(prefix=ints([1])), "causal"),
        (dict(softcap=-1.0), "softcap"),
        (dict(softcap=float("nan")), "softcap"),
        (dict(scale=float("inf")), "scale"),
    ]
    for change, text in bad:
        args = dict(q=q, k=k, v=k)
        args.update(change)
        with pytest.raises(ValueError, match=text):
            attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    assert attention(q, k, k).shape == q.shape


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_reaches_only_what_sees_it(bad, softcap, dim, dtype):
    # in order: queries before the token see nothing of it, the others all of it, element by element
    for n, at, nq in ((150, 100, 150), (70, 69, 70), (300, 290, 20)):
        q, k, v, _ = inputs(nq, n, 4, 2, dim, dtype, n)
        want = A.attention(q, k, v, [0, nq], [0, n], causal=True, softcap=softcap)
        v[at, :, 3::7] = bad
        first = at - (n - nq)  # the first query that sees it
        got = run(q, k, v, None, causal=True, softcap=softcap, offsets=ints([0, nq]), k_offsets=ints([0, n]))
        check({"out": got["out"][:first]}, {"out": tuple(t[:first] for t in want["out"])})
        check({"lse": got["lse"]}, want)
        seen = got["out"][first:].cpu()
        assert not bool(torch.isfinite(seen[..., 3::7]).any())
        clean = [d for d in range(dim) if d % 7 != 3]
        check({"out": seen[..., clean]}, {"out": tuple(t[first:, :, clean] for t in want["out"])})
        # a key: its scores are not finite where it is seen
        q, k, v, _ = inputs(nq, n, 4, 2, dim, dtype, n)
        k[at] = float("nan")
        got = run(q, k, v, None, causal=True, softcap=softcap, offsets=ints([0, nq]), k_offsets=ints([0, n]))
        check({"out": got["out"][:first], "lse": got["lse"][:first]},
              {name: tuple(t[:first] for t in want[name]) for name in ("out", "lse")})
        assert bool(got["out"][first:].isnan().all()) and bool(got["lse"][first:].isnan().all())


def test_captured_in_a_graph():
    """Calls that take workspaces and several launches, replayed with other work between."""
    from amdsplat import clip_grad_norm, rotary_axes

    q, k, v, g = (t.to(DEV) for t in inputs(600, 600, 4, 1, 64, torch.bfloat16, 33))
    one = q[:1].clone()
    x = [torch.randn(5000, device=DEV), torch.randn(77, device=DEV).bfloat16()]
    out = [torch.empty_like(t) for t in x]
    pos = torch.arange(600, device=DEV, dtype=torch.float32)[:, None]

    def work():
        a, b = rotary_axes(q, k, pos, (32,))
        r = run(a, b, v, g, causal=True)
        long = attention(one, k.repeat(20, 1, 1), v.repeat(20, 1, 1), offsets=ints_one, k_offsets=ints_all)
        return [*r.values(), long, clip_grad_norm(x, 1.0, out=out), *out]

    ints_one, ints_all = ints([0, 1]), ints([0, 12000])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = work()
    for i in range(4):
        q.mul_(1.01)
        x[0].add_(0.1)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        for a, b in zip(got, [t.clone() for t in work()]):
            assert torch.equal(a, b), i
        torch.empty(1 << 22, device=DEV).normal_()
