"""Argument checks of the predictor's operators that come before anything touches the GPU: the C entry
points return a GS_ERR_* code with a message, the Python surfaces raise. Only NULL pointers, and made-up
addresses in calls that are refused for an alignment or a size, are passed."""
import ctypes as C
import math

import pytest
import torch

import amdsplat
from amdsplat import _lib

ARG, WORKSPACE, ALIGN = 1, 2, 4


def expect(rc, code, text):
    msg = _lib.lib().gs_last_error().decode()
    assert rc == code, (rc, msg)
    assert text in msg, msg


def attention_args(**kw):
    a = dict(q=256, k=256, v=256, out=256, lse=256, q_tokens=16, k_tokens=16, q_token_stride=256, q_head_stride=64,
             k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, docs=1, heads=4, kv_heads=2,
             dim=64, dtype=_lib.GS_BFLOAT16, causal=0, softcap=0.0, scale=0.125)
    a.update(kw)
    return _lib.GsAttention(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=1), ARG, "dtype"),
    (dict(dtype=7), ARG, "dtype"),
    (dict(heads=3), ARG, "multiple"),
    (dict(kv_heads=0), ARG, "multiple"),
    (dict(heads=0), ARG, "multiple"),
    (dict(dim=0), ARG, "head size"),
    (dict(dim=60), ARG, "head size"),
    (dict(dim=136), ARG, "head size"),
    (dict(docs=0), ARG, "document"),
    (dict(docs=2), ARG, "offsets"),
    (dict(q_tokens=-1), ARG, "token counts"),
    (dict(k_tokens=1 << 30), ARG, "too many"),
    (dict(prefix=256), ARG, "prefix"),
    (dict(softcap=-1.0), ARG, "softcap"),
    (dict(softcap=math.inf), ARG, "softcap"),
    (dict(scale=math.nan), ARG, "scale"),
    (dict(q=None), ARG, "null"),
    (dict(lse=None), ARG, "null"),
    (dict(v=None), ARG, "null"),
    (dict(k_token_stride=129), ALIGN, "strides"),
    (dict(v_head_stride=-64), ALIGN, "strides"),
    (dict(q_token_stride=1 << 22), ALIGN, "strides"),
    (dict(k=264), ALIGN, "aligned"),
    (dict(out=258), ALIGN, "aligned"),
])
def test_attention_arguments(kw, code, text):
    L = _lib.lib()
    a = attention_args(**kw)
    expect(L.gs_attention_fwd(C.byref(a), None, 0, None), code, text)
    expect(L.gs_attention_bwd(C.byref(a), 256, 256, 256, 256, 256, 1 << 20, None), code, text)


def test_attention_calls():
    L = _lib.lib()
    a = attention_args()
    expect(L.gs_attention_fwd(None, None, 0, None), ARG, "NULL")
    expect(L.gs_attention_bwd(C.byref(a), None, 256, 256, 256, 256, 1 << 20, None), ARG, "null")
    expect(L.gs_attention_bwd(C.byref(a), 256, 256, None, 256, 256, 1 << 20, None), ARG, "null")
    expect(L.gs_attention_bwd(C.byref(a), 258, 256, 256, 256, 256, 1 << 20, None), ALIGN, "aligned")
    need = L.gs_attention_bwd_workspace_size(C.byref(a))
    expect(L.gs_attention_bwd(C.byref(a), 256, 256, 256, 256, 256, need - 1, None), WORKSPACE, "workspace")
    expect(L.gs_attention_bwd(C.byref(a), 256, 256, 256, 256, None, need, None), WORKSPACE, "workspace")
    assert L.gs_attention_bwd_workspace_size(None) == 0 and L.gs_attention_fwd_workspace_size(None) == 0


def rotary_args(sections=(8, 8), **kw):
    a = dict(q=256, q_out=256, positions=256, tokens=4, q_token_stride=128, q_head_stride=64, base=100.0, q_heads=2,
             dim=64, axes=2, dtype=_lib.GS_FLOAT32)
    a.update(kw)
    r = _lib.GsRotary(**a)
    r.sections[:len(sections)] = sections
    return r


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=1), ARG, "dtype"),
    (dict(axes=0), ARG, "axes"),
    (dict(axes=5), ARG, "axes"),
    (dict(tokens=-1), ARG, "count"),
    (dict(q_heads=0), ARG, "count"),
    (dict(base=0.0), ARG, "base"),
    (dict(base=math.nan), ARG, "base"),
    (dict(sections=(-1, 8)), ARG, "section"),
    (dict(sections=(20, 20)), ARG, "do not fit"),
    (dict(sections=(0, 0)), ARG, "do not fit"),
    (dict(positions=None), ARG, "null"),
    (dict(q_out=None), ARG, "null"),
    (dict(k_heads=2), ARG, "null"),
    (dict(q=257), ALIGN, "misaligned"),
])
def test_rotary_arguments(kw, code, text):
    expect(_lib.lib().gs_rotary_axes(C.byref(rotary_args(**kw)), None), code, text)
    expect(_lib.lib().gs_rotary_axes(None, None), ARG, "NULL")


def test_gradient_tables():
    L = _lib.lib()
    ptrs, sizes, types = (C.c_uint64 * 2)(256, 512), (C.c_int64 * 2)(10, 20000), (C.c_int32 * 2)(0, 2)
    need = L.gs_grad_norm_workspace_size(sizes, 2)
    assert need >= 16 and need % 8 == 0 and L.gs_grad_norm_workspace_size(None, 2) == 0
    norm = lambda p=ptrs, s=sizes, t=types, n=2, m=1.0, o=256, c=260, w=256, b=need: L.gs_grad_norm(  # noqa: E731
        p, s, t, n, m, o, c, w, b, None)
    expect(norm(n=-1), ARG, "negative")
    expect(norm(p=None), ARG, "null")
    expect(norm(s=(C.c_int64 * 2)(10, -1)), ARG, "size")
    expect(norm(t=(C.c_int32 * 2)(0, 1)), ARG, "dtype")
    expect(norm(p=(C.c_uint64 * 2)(0, 512)), ARG, "null")
    expect(norm(p=(C.c_uint64 * 2)(258, 512)), ALIGN, "misaligned")
    expect(norm(o=None), ARG, "null")
    expect(norm(m=-1.0), ARG, "max_norm")
    expect(norm(m=math.nan), ARG, "max_norm")
    expect(norm(b=need - 1), WORKSPACE, "workspace")
    expect(norm(w=None), WORKSPACE, "workspace")
    expect(norm(w=260), ALIGN, "misaligned")
    scale = lambda p=ptrs, o=ptrs, c=256: L.gs_grad_scale(p, o, sizes, types, 2, c, None)  # noqa: E731
    expect(scale(c=None), ARG, "null")
    expect(scale(o=None), ARG, "null")
    expect(scale(o=(C.c_uint64 * 2)(256, 0)), ARG, "NULL")
    expect(scale(o=(C.c_uint64 * 2)(256, 513)), ALIGN, "misaligned")
    expect(scale(c=257), ALIGN, "misaligned")
    group = (_lib.GsAdamGroup * 1)()
    expect(L.gs_adam_step_scaled(group, 1, 0, None, None, None), ARG, "factor")
    expect(L.gs_adam_step_scaled(group, 1, 0, None, 258, None), ARG, "factor")


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(4, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        amdsplat.attention(x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        amdsplat.rotary_axes(x, None, torch.zeros(4, 1), (8,))
    with pytest.raises(ValueError, match="GPU"):
        amdsplat.grad_norm([x])
    with pytest.raises(ValueError, match="GPU"):
        amdsplat.clip_grad_norm([x], 1.0)
