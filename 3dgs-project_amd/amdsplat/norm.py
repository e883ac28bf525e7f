"""Norms before and after a transformer block on the GPU (gs_residual_norm_fwd / gs_residual_norm_bwd).

`norm(x, weight)` is an RMS or layer norm over the last dimension. `residual_norm(x, y, weight, ...)` is what
lies between two blocks, in one launch each way: the block's output y is normed, dropped out, gated and added to
the residual stream x, and the sum is normed for the next block. The stream may be float32 beside
bfloat16 blocks. Statistics and sums are float32.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._grad import tracked
from ._lib import call_on, ptr
from .dropout import check_rule

MAX_WIDTH = 8192  # GS_NORM_MAX_WIDTH
_DTYPES = {torch.float32: _lib.GS_FLOAT32, torch.bfloat16: _lib.GS_BFLOAT16}


def _rows(t):
    return t if t is None or ((t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0) else t.contiguous()


def _args(x, y, weight, bias, post_weight, post_bias, gate, seed_at, h, n, stats, rule) -> _lib.GsResidualNorm:
    layer, eps, scale, p, seed, draw, n_dtype = rule
    w = weight if weight is not None else bias if bias is not None else post_weight  # (there is no post bias without it)
    token = gate is not None and gate.dim() == 2
    rows, width = x.shape
    return _lib.GsResidualNorm(
        x.data_ptr(), None if y is None else y.data_ptr(), None if weight is None else weight.data_ptr(),
        None if bias is None else bias.data_ptr(), None if post_weight is None else post_weight.data_ptr(),
        None if post_bias is None else post_bias.data_ptr(), None if gate is None else gate.data_ptr(),
        None if h is None else h.data_ptr(), None if n is None else n.data_ptr(),
        None if stats is None else stats.data_ptr(), None if seed_at is None else seed_at.data_ptr(), seed, draw, rows,
        x.stride(0), 0 if y is None else y.stride(0), gate.stride(0) if token else 0, p, eps, scale, width,
        _DTYPES[x.dtype], _DTYPES[n_dtype], 0 if w is None else _DTYPES[w.dtype],
        0 if gate is None else _DTYPES[gate.dtype], token, layer)


def _forward(x, y, weight, bias, post_weight, post_bias, gate, seed_at, rule, keep: bool):
    shape, device = x.shape, x.device
    h = None if y is None else torch.empty(shape, dtype=x.dtype, device=device)
    n = torch.empty(shape, dtype=rule[-1], device=device)
    stats = torch.empty((shape[0], 4), dtype=torch.float32, device=device) if keep else None
    a = _args(x, y, weight, bias, post_weight, post_bias, gate, seed_at, h, n, stats, rule)
    call_on(device, "gs_residual_norm_fwd", C.byref(a))
    return h, n, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, bias, post_weight, post_bias, gate, seed_at, rule):
        h, n, stats = _forward(x, y, weight, bias, post_weight, post_bias, gate, seed_at, rule, True)
        ctx.save_for_backward(x, y, weight, bias, post_weight, post_bias, gate, seed_at, stats)
        ctx.rule = rule
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_h, d_n):
        if d_h is None and d_n is None:
            return (None,) * 9
        x, y, *weights, gate, seed_at, stats = ctx.saved_tensors
        d_h, d_n = (None if t is None else t.contiguous() for t in (d_h, d_n))
        outs = [torch.empty_like(t, memory_format=torch.contiguous_format) if need and t is not None else None
                for t, need in zip((x, y, *weights, gate), ctx.needs_input_grad)]
        a = _args(x, y, *weights, gate, seed_at, None, None, stats, ctx.rule)
        size = _lib.size_call("gs_residual_norm_bwd_workspace_size", C.byref(a))
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
        call_on(x.device, "gs_residual_norm_bwd", C.byref(a), ptr(d_h), ptr(d_n), *map(ptr, outs), ws.data_ptr(), size)
        return (*outs, None, None)


def _vector(t, name: str, width: int, device, dtype=None):
    if t is None:
        return None
    if t.shape != (width,) or t.dtype not in _DTYPES or t.device != device or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be [{width}], float32 or bfloat16 like the other weights, on the tensors' device")
    return t if t.is_contiguous() else t.contiguous()


def _rule(x, kind: str, eps, dtype):
    if x.dim() != 2:
        raise ValueError("the rows must be [tokens, width]")
    if x.dtype not in _DTYPES:
        raise ValueError(f"float32 or bfloat16 rows, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError("the rows must be on the GPU")
    if not 1 <= x.shape[1] <= MAX_WIDTH:
        raise ValueError(f"width {x.shape[1]}: 1 to {MAX_WIDTH} are provided")
    if kind not in ("rms", "layer"):
        raise ValueError('kind must be "rms" or "layer"')
    eps = float(eps)
    if not 0.0 < C.c_float(eps).value <= 1e30:
        raise ValueError("eps must be positive and finite in float32")
    if dtype not in _DTYPES or (x.dtype == torch.bfloat16 and dtype != torch.bfloat16):
        raise ValueError(f"a {x.dtype} stream does not go with {dtype}: float32 streams take float32 or bfloat16, "
                         "bfloat16 streams bfloat16")
    return kind == "layer", eps


def norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, kind: str = "rms",
         eps: float = 1e-6, dtype: torch.dtype | None = None) -> torch.Tensor:
    """weight x^ + bias over the rows of x [T, C], x^ = x / sqrt(mean x^2 + eps), or with kind "layer"
    (x - mean x) / sqrt(var x + eps); differentiable in x, weight and bias ([C], one dtype, either may be None). dtype
    of the result: x's by default, or bfloat16 of a float32 x. C up to 8192, T below 2^31, T C below 2^38; the mean of a
    row's squares has to be finite in float32. No forward-mode derivative."""
    dtype = x.dtype if dtype is None else dtype
    layer, eps = _rule(x, kind, eps, dtype)
    weight = _vector(weight, "weight", x.shape[1], x.device)
    bias = _vector(bias, "bias", x.shape[1], x.device, None if weight is None else weight.dtype)
    args = (_rows(x), None, weight, bias, None, None, None, None, (layer, eps, 1.0, 0.0, 0, 0, dtype))
    return (_ResidualNorm.apply(*args) if tracked(x, weight, bias) else _forward(*args, False))[1]


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, kind: str = "rms", eps: float = 1e-6,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, dropout: float = 0.0, seed=None, draw: int = 0):
    """(h, n) of the residual stream x [T, C] and a block's output y [T, C]:

        b = y, or with post_weight: y normed, times post_weight (+ post_bias)
        h = x + scale * gate * dropout(b)        n = h normed, times weight (+ bias)

    h has x's dtype and n y's: float32 streams take float32 or bfloat16 blocks, bfloat16 streams bfloat16 ones.
    kind, eps: of both norms, as in `norm`, and so are the limits. weight, bias, post_weight, post_bias: [C] of one
    dtype. gate: [C] or [T, C]. dropout, seed, draw: as in `dropout`, for the rows of y. h enters n unrounded.
    Differentiable in all tensors, through h and n; gradients of [C] tensors are summed in float32 in a fixed order. Nothing
    but the inputs and four numbers a row is kept for the backward pass. No forward-mode derivative."""
    if x.dim() != 2 or x.shape != y.shape:
        raise ValueError(f"x and y must be [tokens, width] alike, got {tuple(x.shape)} and {tuple(y.shape)}")
    if y.device != x.device:
        raise ValueError("x and y must be on one GPU")
    layer, eps = _rule(x, kind, eps, y.dtype)
    width, device = x.shape[1], x.device
    w = weight if weight is not None else bias if bias is not None else post_weight if post_weight is not None else post_bias
    if w is not None:
        dtype = w.dtype
        weight = None if weight is None else _vector(weight, "weight", width, device, dtype)
        bias = None if bias is None else _vector(bias, "bias", width, device, dtype)
        post_weight = None if post_weight is None else _vector(post_weight, "post_weight", width, device, dtype)
        post_bias = None if post_bias is None else _vector(post_bias, "post_bias", width, device, dtype)
    if post_bias is not None and post_weight is None:
        raise ValueError("post_bias without post_weight")
    if gate is not None:
        if gate.shape not in ((width,), tuple(x.shape)) or gate.dtype not in _DTYPES or gate.device != device:
            raise ValueError(f"gate must be [{width}] or {list(x.shape)}, float32 or bfloat16, on the tensors' device")
        gate = gate if gate.dim() == 1 and gate.is_contiguous() else _rows(gate) if gate.dim() == 2 else gate.contiguous()
    scale = float(scale)
    if not math.isfinite(C.c_float(scale).value):
        raise ValueError("scale must be finite in float32")
    p, seed_at, seed, draw = check_rule(dropout, seed, draw, device)
    args = (_rows(x), _rows(y), weight, bias, post_weight, post_bias, gate, seed_at,
            (layer, eps, scale, p, seed, draw, y.dtype))
    if tracked(x, y, weight, bias, post_weight, post_bias, gate):
        return _ResidualNorm.apply(*args)
    return _forward(*args, False)[:2]
