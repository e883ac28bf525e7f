"""Argument checks of the block operators' C entry points that come before anything touches the GPU. Only NULL
pointers, and made-up addresses in calls that are refused for an alignment or a size, are passed."""
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


def norm_args(**kw):
    a = dict(x=256, y=256, weight=256, bias=256, post_weight=256, post_bias=256, gate=256, h=256, n=256, stats=256,
             rows=4, x_stride=64, y_stride=64, gate_stride=64, eps=1e-6, scale=1.0, width=64)
    a.update(kw)
    return _lib.GsResidualNorm(**a)


BF = _lib.GS_BFLOAT16


@pytest.mark.parametrize("kw,code,text", [
    (dict(x_dtype=1), ARG, "dtypes"), (dict(y_dtype=7), ARG, "dtypes"), (dict(x_dtype=BF), ARG, "bfloat16 stream"),
    (dict(weight_dtype=1), ARG, "weight dtype"), (dict(gate_dtype=1), ARG, "gate dtype"), (dict(rows=-1), ARG, "row count"),
    (dict(rows=1 << 31), ARG, "row count"), (dict(width=0), ARG, "width"), (dict(width=8193), ARG, "width"),
    (dict(eps=0.0), ARG, "eps"), (dict(eps=math.inf), ARG, "eps"), (dict(eps=math.nan), ARG, "eps"),
    (dict(scale=math.nan), ARG, "scale"), (dict(scale=math.inf), ARG, "scale"), (dict(dropout=1.0), ARG, "dropout"),
    (dict(dropout=-0.1), ARG, "dropout"), (dict(dropout=math.nan), ARG, "dropout"), (dict(y=None), ARG, "needs y"),
    (dict(post_weight=None), ARG, "post bias"), (dict(x=None), ARG, "null"), (dict(x=257), ALIGN, "misaligned"),
    (dict(y_dtype=BF, y=257), ALIGN, "misaligned"), (dict(weight=258), ALIGN, "misaligned"),
    (dict(stats=264), ALIGN, "misaligned"), (dict(seed_at=260), ALIGN, "misaligned"),
])
def test_norm_arguments(kw, code, text):
    L = _lib.lib()
    a = norm_args(**kw)
    expect(L.gs_residual_norm_fwd(C.byref(a), None), code, text)
    expect(L.gs_residual_norm_bwd(C.byref(a), *[256] * 10, 1 << 30, None), code, text)


def test_norm_calls():
    L = _lib.lib()
    a = norm_args()
    need = L.gs_residual_norm_bwd_workspace_size(C.byref(a))
    back = lambda a, dh=256, dx=256, dy=256, dpw=256, dg=256, ws=256, n=need: L.gs_residual_norm_bwd(  # noqa: E731
        C.byref(a), dh, 256, dx, dy, 256, 256, dpw, 256, dg, ws, n, None)
    expect(L.gs_residual_norm_fwd(None, None), ARG, "NULL")
    expect(L.gs_residual_norm_fwd(C.byref(norm_args(rows=(1 << 31) - 1, width=8192)), None), ARG, "too many")
    expect(L.gs_residual_norm_fwd(C.byref(norm_args(n=None)), None), ARG, "null")
    expect(L.gs_residual_norm_fwd(C.byref(norm_args(h=None)), None), ARG, "null")
    expect(back(norm_args(stats=None)), ARG, "statistics")
    expect(back(a, n=need - 1), WORKSPACE, "workspace")
    expect(back(a, ws=None), WORKSPACE, "workspace")
    expect(back(a, ws=264), ALIGN, "misaligned")
    expect(back(a, dx=258), ALIGN, "misaligned")
    alone = dict(y=None, gate=None, post_weight=None, post_bias=None)
    expect(back(norm_args(**alone)), ARG, "not there")
    expect(back(norm_args(gate=None)), ARG, "not there")
    expect(back(norm_args(post_weight=None, post_bias=None)), ARG, "not there")
    assert L.gs_residual_norm_bwd_workspace_size(None) == 0


def test_dropout_arguments():
    L = _lib.lib()
    drop = lambda x=256, out=256, rows=4, width=64, dtype=0, p=0.5, at=None: L.gs_dropout(  # noqa: E731
        x, out, rows, 64, width, dtype, p, at, 1, 0, None)
    expect(drop(dtype=1), ARG, "dtype")
    expect(drop(rows=-1), ARG, "size")
    expect(drop(rows=1 << 32), ARG, "size")
    expect(drop(width=-1), ARG, "size")
    expect(drop(p=1.0), ARG, "p must")
    expect(drop(p=math.nan), ARG, "p must")
    expect(drop(x=None), ARG, "null")
    expect(drop(out=None), ARG, "null")
    expect(drop(x=258), ALIGN, "misaligned")
    expect(drop(at=260), ALIGN, "misaligned")
    expect(drop(rows=(1 << 32) - 1, width=1 << 20), ARG, "too many")
    assert drop(rows=0) == 0 and drop(width=0, x=None) == 0


def scan_args(**kw):
    a = dict(x=256, forget=256, gate=256, initial=256, y=256, state=256, carry=256, offsets=256, tokens=400, x_stride=64,
             forget_stride=64, gate_stride=64, docs=3, width=64)
    a.update(kw)
    return _lib.GsGatedScan(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=1), ARG, "dtype"), (dict(tokens=-1), ARG, "token count"), (dict(tokens=1 << 31), ARG, "token count"),
    (dict(width=0), ARG, "width"), (dict(width=(1 << 20) + 1), ARG, "width"), (dict(docs=0), ARG, "document"),
    (dict(docs=1 << 30), ARG, "document"), (dict(tokens=1 << 30, width=1 << 12), ARG, "too many"), (dict(offsets=None), ARG, "offsets"), (dict(x=None), ARG, "null"),
    (dict(forget=None), ARG, "null"), (dict(x=258), ALIGN, "misaligned"), (dict(state=258), ALIGN, "misaligned"),
    (dict(offsets=258), ALIGN, "misaligned"), (dict(dtype=BF, gate=257), ALIGN, "misaligned"),
])
def test_scan_arguments(kw, code, text):
    L = _lib.lib()
    a = scan_args(**kw)
    expect(L.gs_gated_scan_fwd(C.byref(a), 256, 1 << 30, None), code, text)
    expect(L.gs_gated_scan_bwd(C.byref(a), *[256] * 7, 1 << 30, None), code, text)


def test_scan_calls():
    L = _lib.lib()
    a = scan_args()
    need = L.gs_gated_scan_workspace_size(400, 64)
    assert need > 0 and L.gs_gated_scan_workspace_size(0, 64) == 0 and L.gs_gated_scan_chunks(-1) == 0
    expect(L.gs_gated_scan_fwd(None, None, 0, None), ARG, "NULL")
    expect(L.gs_gated_scan_fwd(C.byref(a), 256, need - 1, None), WORKSPACE, "workspace")
    expect(L.gs_gated_scan_fwd(C.byref(a), None, need, None), WORKSPACE, "workspace")
    expect(L.gs_gated_scan_fwd(C.byref(a), 264, need, None), ALIGN, "misaligned")
    expect(L.gs_gated_scan_fwd(C.byref(scan_args(y=None)), 256, need, None), ARG, "null")
    back = lambda a, dy=256, ds=256, dx=256, dg=256: L.gs_gated_scan_bwd(  # noqa: E731
        C.byref(a), dy, ds, dx, 256, dg, 256, 256, need, None)
    expect(back(scan_args(carry=None)), ARG, "carried")
    expect(back(a, dy=None), ARG, "carried")
    expect(back(scan_args(gate=None)), ARG, "not there")
    expect(back(a, dx=258), ALIGN, "misaligned")
    expect(back(a, ds=258), ALIGN, "misaligned")


def linear_args(**kw):
    a = dict(x=256, weight=256, bias=256, residual=256, out=256, z=256, rows=100, x_stride=64, weight_stride=64,
             residual_stride=40, inputs=64, outputs=40, activation=2)
    a.update(kw)
    return _lib.GsLinear(**a)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=1), ARG, "dtypes"), (dict(out_dtype=1), ARG, "dtypes"), (dict(out_dtype=BF), ARG, "float32 products"),
    (dict(bias_dtype=1), ARG, "bias dtype"), (dict(z_dtype=1), ARG, "z must"), (dict(z_dtype=BF), ARG, "z must"),
    (dict(activation=-1), ARG, "activation"), (dict(activation=5), ARG, "activation"), (dict(rows=-1), ARG, "row count"),
    (dict(rows=1 << 31), ARG, "row count"), (dict(inputs=0), ARG, "inputs"), (dict(inputs=(1 << 19) + 4), ARG, "inputs"),
    (dict(outputs=0), ARG, "outputs"), (dict(x=None), ARG, "null"), (dict(weight=None), ARG, "null"),
    (dict(x_stride=66), ALIGN, "strides"), (dict(weight_stride=-64), ALIGN, "strides"), (dict(x_stride=1 << 20), ALIGN, "strides"),
    (dict(x=260), ALIGN, "misaligned"), (dict(weight=264), ALIGN, "misaligned"), (dict(bias=258), ALIGN, "misaligned"),
    (dict(rows=(1 << 31) - 1, outputs=1 << 19), ARG, "too many"),
])
def test_linear_arguments(kw, code, text):
    L = _lib.lib()
    a = linear_args(**kw)
    expect(L.gs_linear_fwd(C.byref(a), 256, 1 << 62, None), code, text)
    expect(L.gs_linear_bwd(C.byref(a), 256, 256, 256, 256, 256, 1 << 62, None), code, text)


def test_linear_calls():
    L = _lib.lib()
    # few rows are read at any address, but for gradients
    expect(L.gs_linear_fwd(C.byref(linear_args(rows=16, x=260, x_stride=65, weight=258)), None, 0, None), ALIGN, "misaligned")
    expect(L.gs_linear_bwd(C.byref(linear_args(rows=16, x=260)), 256, 256, 256, 256, 256, 1 << 62, None), ALIGN, "misaligned")
    rows = lambda **kw: _lib.GsRows(**{**dict(src=256, dst=256, rows=4, cols=60, src_stride=70, dst_stride=64), **kw})  # noqa: E731
    pack = lambda n=2, dtype=0, **kw: L.gs_rows_pack((_lib.GsRows * 2)(rows(), rows(**kw)), n, dtype, None)  # noqa: E731
    expect(pack(dtype=1), ARG, "dtype")
    expect(pack(n=3), ARG, "two sets")
    expect(L.gs_rows_pack(None, 1, 0, None), ARG, "two sets")
    expect(pack(rows=-1), ARG, "size")
    expect(pack(dst_stride=60), ARG, "size")
    expect(pack(dst_stride=56), ARG, "size")
    expect(pack(src=None), ARG, "null")
    expect(pack(dst=264), ALIGN, "misaligned")
    expect(pack(src=258), ALIGN, "misaligned")
    expect(pack(rows=1 << 31, dst_stride=1 << 10), ARG, "too many")
    assert L.gs_rows_pack(None, 0, 0, None) == 0
    a = linear_args()
    need = L.gs_linear_bwd_workspace_size(C.byref(a))
    assert need > 0 and L.gs_linear_bwd_workspace_size(None) == 0 and L.gs_linear_fwd_workspace_size(None) == 0
    back = lambda a, d=256, dx=256, ws=256, n=need: L.gs_linear_bwd(C.byref(a), d, dx, 256, 256, ws, n, None)  # noqa: E731
    expect(L.gs_linear_fwd(None, None, 0, None), ARG, "NULL")
    expect(L.gs_linear_fwd(C.byref(linear_args(out=None)), 256, 1 << 40, None), ARG, "null")
    expect(L.gs_linear_fwd(C.byref(linear_args(out=258)), 256, 1 << 40, None), ALIGN, "misaligned")
    expect(back(a, d=None), ARG, "null")
    expect(back(linear_args(z=None)), ARG, "needs z")
    expect(back(a, n=need - 1), WORKSPACE, "workspace")
    expect(back(a, ws=None), WORKSPACE, "workspace")
    expect(back(a, ws=264), ALIGN, "misaligned")
    expect(back(a, d=264), ALIGN, "misaligned")
    expect(back(a, dx=258), ALIGN, "misaligned")
    split = linear_args(rows=64, inputs=8192, outputs=64, x_stride=8192, weight_stride=8192)
    need = L.gs_linear_fwd_workspace_size(C.byref(split))
    assert need > 0
    expect(L.gs_linear_fwd(C.byref(split), 256, need - 1, None), WORKSPACE, "workspace")
    expect(L.gs_linear_fwd(C.byref(split), 264, need, None), ALIGN, "misaligned")


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(4, 16)
    for call in (lambda: amdsplat.norm(x), lambda: amdsplat.residual_norm(x, x), lambda: amdsplat.dropout(x, 0.5, 1),
                 lambda: amdsplat.gated_scan(x, x), lambda: amdsplat.linear(x, x)):
        with pytest.raises(ValueError, match="GPU"):
            call()
