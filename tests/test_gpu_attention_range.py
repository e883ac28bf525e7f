"""GPU parity of amdsplat.attention at the ends of what its arguments may be: large and small values under
capped scores, large and small caps and scales. Values and bounds are the float64 oracle's
(oracle/attention_ref.py)."""
import pytest
import torch

import attention_ref as A
from test_gpu_attention import DT, check, inputs, ints, run

pytestmark = pytest.mark.gpu


def aligned(nq, nk, signs, size, dtype, seed, dim=64, heads=4, kv_heads=2):
    """Queries and keys whose scores before the cap are near signs[j] * size: each is a fixed pattern of +-1 with
    an eighth of noise."""
    g = torch.Generator().manual_seed(seed)
    pattern = torch.randint(0, 2, (dim,), generator=g) * 2.0 - 1.0
    a = (size / dim ** 0.5) ** 0.5  # a^2 dim / sqrt(dim) = size
    noise = lambda *s: 1.0 + 0.125 * torch.randn(*s, generator=g)  # noqa: E731
    q = (a * pattern * noise(nq, heads, dim)).to(dtype)
    k = (a * signs[:, None, None] * pattern * noise(nk, kv_heads, dim)).to(dtype)
    return q, k, torch.randn(nk, kv_heads, dim, generator=g)


SIGNS = {
    "top": lambda n: torch.ones(n),
    "bottom": lambda n: -torch.ones(n),
    "rising": lambda n: torch.where(torch.arange(n) < n - n // 3, -1.0, 1.0),
    "falling": lambda n: torch.where(torch.arange(n) < n // 3, 1.0, -1.0),
}


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("signs", SIGNS)
@pytest.mark.parametrize("softcap", [15.0, 30.0, 50.0, 62.0, 100.0])
@pytest.mark.parametrize("gain", [1e30, 1e-25])
@pytest.mark.parametrize("nq,nk,causal", [(150, 150, True), (150, 150, False), (1, 9000, False), (3, 4000, True),
                                          (181, 5000, True)])
def test_values_of_every_size_under_a_cap(nq, nk, causal, gain, softcap, signs, dtype):
    """Saturated scores at either end of the cap: the output is a mean of the values whatever their size. The
    sums stay in float32's range (1e30 times 2^8 times 9000 keys)."""
    q, k, v = aligned(nq, nk, SIGNS[signs](nk), 10 * softcap, dtype, nk + nq)
    v = (gain * v).to(dtype)
    got = run(q, k, v, None, causal=causal, softcap=softcap, offsets=ints([0, nq]), k_offsets=ints([0, nk]))
    check(got, A.attention(q, k, v, [0, nq], [0, nk], causal=causal, softcap=softcap))
    assert bool(got["out"].any())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("softcap", [257.0, 300.0, 1e4, 1e6, 1e8])
@pytest.mark.parametrize("nq,nk,causal,train", [(150, 150, True, True), (97, 97, False, True), (1, 3000, False, False),
                                                (130, 4000, True, False)])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_scores_far_below_the_cap(dim, nq, nk, causal, train, softcap, dtype):
    """A cap far above the scores changes them little, and its size is no error of theirs. The bound is the one
    of uncapped scores, with 4 units of 2^-23 of the scores more for the tanh (two operations beside the D + 4 of the
    product): (D + 8) / (D + 4) of it."""
    q, k, v, g = inputs(nq, nk, 4, 2, dim, dtype, dim + nk)
    at = ([0, nq], [0, nk])
    d_out = g if train else None
    got = run(q, k, v, d_out, causal=causal, softcap=softcap, offsets=ints(at[0]), k_offsets=ints(at[1]))
    want = A.attention(q, k, v, *at, causal=causal, softcap=softcap, d_out=d_out)
    near = A.attention(q, k, v, *at, causal=causal, d_out=d_out)
    check(got, {n: (want[n][0], near[n][1] * (dim + 8) / (dim + 4)) for n in want})


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("softcap", [2.0 ** -96, 1e-20, 1e-3, 2.0 ** 96])
def test_caps_at_their_ends(softcap, dtype):
    """Under a cap of next to nothing every key counts the same and the scores have next to no gradient (a slope times
    the scale); under one far above the scores nothing is capped. A key of zeros has a score of 0."""
    nq = nk = 150
    q, k, v, g = inputs(nq, nk, 4, 2, 64, dtype, 41)
    k[7] = 0.0
    at = ([0, nq], [0, nk])
    got = run(q, k, v, g, causal=True, softcap=softcap, offsets=ints(at[0]), k_offsets=ints(at[1]))
    want = A.attention(q, k, v, *at, causal=True, softcap=softcap, d_out=g)
    near = A.attention(q, k, v, *at, causal=True, d_out=g)
    check(got, {n: (want[n][0], torch.maximum(want[n][1], near[n][1] * 72 / 68) if softcap < 1 else near[n][1] * 72 / 68)
                for n in want})


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -50, 2.0 ** 50, 2.0 ** 61])
def test_scales_of_every_size(size, causal, dtype):
    """Queries and keys of one size, and the scale that takes it off again: the scores are those of size 1, since a
    power of two changes no rounding. Gradients are then of the other size, hence of the oracle's as well."""
    for nq, nk in ((150, 150), (1, 700)):
        q, k, v, g = inputs(nq, nk, 4, 2, 64, dtype, 43)
        at, scale = ([0, nq], [0, nk]), 0.125 / size ** 2
        d_out = g if nq > 1 else None
        got = run(q * size, k * size, v, d_out, causal=causal, scale=scale, offsets=ints(at[0]), k_offsets=ints(at[1]))
        check(got, A.attention(q * size, k * size, v, *at, causal=causal, scale=scale, d_out=d_out))
