"""Caps and scales of attention that are refused before anything touches the GPU, and the ends of what is not: the
calls below pass made-up addresses, and those that are accepted stop at the missing workspace."""
import ctypes as C

import pytest
import torch

from amdsplat import _lib, attention
from test_operator_errors import ARG, WORKSPACE, attention_args, expect


def refused(text, **kw):
    a = attention_args(**kw)
    expect(_lib.lib().gs_attention_fwd(C.byref(a), None, 0, None), ARG, text)
    expect(_lib.lib().gs_attention_bwd(C.byref(a), 256, 256, 256, 256, 256, 1 << 20, None), ARG, text)


def accepted(**kw):
    a = attention_args(**kw)
    expect(_lib.lib().gs_attention_bwd(C.byref(a), 256, 256, 256, 256, None, 0, None), WORKSPACE, "workspace")


def python(text, **kw):
    # (tensors of the meta device that claim to be on the GPU, so that the checks behind that one are reached)
    class Fake(torch.Tensor):
        is_cuda = True

    x = torch.empty(4, 2, 16, device="meta").as_subclass(Fake)
    with pytest.raises(ValueError, match=text):
        attention(x, x, x, **kw)


@pytest.mark.parametrize("softcap", [1e-46, 1e-40, 2.0 ** -97, 2.0 ** 97, 1e39])
def test_caps_out_of_range(softcap):
    """1e-46 is 0 in float32, where 0 means no cap; a smaller cap than 2^-96 makes scale / cap infinite, and a
    score of 0 over it NaN; over a larger one than 2^96 ordinary scores underflow."""
    if 0.0 < C.c_float(softcap).value < float("inf"):
        refused("softcap", softcap=softcap)
    python("softcap", softcap=softcap)


@pytest.mark.parametrize("scale,softcap", [(2.0 ** 60, 2.0 ** -66), (-(2.0 ** 60), 2.0 ** -66), (2.0 ** -40, 2.0 ** 87)])
def test_scales_far_from_the_cap(scale, softcap):
    refused("scale / softcap", scale=scale, softcap=softcap)
    python("scale / softcap", scale=scale, softcap=softcap)


@pytest.mark.parametrize("scale", [1e-46, 1e-39, -1e-39, 2.0 ** 127, -(2.0 ** 127), 1e300])
def test_scales_out_of_range(scale):
    if 0.0 < abs(C.c_float(scale).value) < float("inf"):
        refused("scale", scale=scale)
    python("scale", scale=scale)


def test_the_ends_are_accepted():
    for softcap, scale in ((2.0 ** -96, 2.0 ** 29), (2.0 ** -96, 0.125), (2.0 ** 96, 2.0 ** -30), (2.0 ** 96, -8.0),
                           (2.0 ** -96, 0.0), (0.0, 0.0), (30.0, 0.0),
                           (0.0, 2.0 ** -126), (0.0, -(2.0 ** 126))):
        accepted(softcap=softcap, scale=scale)


def test_rows_of_the_output_gradient():
    """The key gradients address 64 rows of d_out with 32 bits. Its tokens are heads * dim apart even where q's are
    not (a broadcast q), so that q's strides do not bound them."""
    wide = dict(q_token_stride=0, q_head_stride=0, k_token_stride=0, k_head_stride=0, v_token_stride=0, v_head_stride=0)
    for heads, kv_heads, dim in ((1 << 16, 1 << 16, 64), (1 << 15, 1 << 15, 128), (1 << 26, 1 << 18, 128)):
        a = attention_args(heads=heads, kv_heads=kv_heads, dim=dim, **wide)
        expect(_lib.lib().gs_attention_bwd(C.byref(a), 256, 256, 256, 256, None, 0, None), ARG, "too many heads")
    accepted(heads=31000, kv_heads=31000, dim=128, **wide)
