"""Projections with their epilogue on the GPU (gs_linear_fwd / gs_linear_bwd).

`linear(x, weight, bias, activation=..., residual=...)` is act(x W^T + b) + residual in one pass over the result: the
halves of a transformer block's MLP and the projections beside attention. bfloat16 products may be added to a
float32 residual stream without being rounded first.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._grad import tracked
from ._lib import call_on, ptr

MAX_WIDTH, FEW_ROWS = 1 << 19, 16  # GS_LINEAR_MAX_WIDTH, GS_LINEAR_FEW_ROWS
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}  # GS_ACT_*
_DTYPES = {torch.float32: (_lib.GS_FLOAT32, 4, 4), torch.bfloat16: (_lib.GS_BFLOAT16, 8, 2)}  # code, elements of 16 bytes, bytes


def _rows(t):
    """t, or a copy whose last dimension is contiguous."""
    return t if t is None or ((t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0) else t.contiguous()


def _ready(t: torch.Tensor, few: bool) -> bool:
    """The kernels can read t through its row stride: the tile kernels where its address, row stride and row length are
    multiples of 16 bytes, a forward of few rows at any."""
    s = t.stride(0)
    if t.shape[0] == 0 or not 0 <= s < 1 << 20:
        return t.shape[0] == 0
    per = _DTYPES[t.dtype][1]
    return few or (t.shape[1] % per == 0 and t.stride(1) == 1 and s % per == 0 and t.data_ptr() % 16 == 0)


def _overlaps(t: torch.Tensor) -> bool:
    return t.shape[0] > 1 and t.stride(0) < t.shape[1]


def _pack(x, weight, few: bool, apart: bool = False):
    """Which of x and weight the kernels cannot read, and None or a buffer with these as rows with zeros behind them. apart:
    rows that overlap are among these."""
    away = (not _ready(x, few) or (apart and _overlaps(x)), not _ready(weight, few) or (apart and _overlaps(weight)))
    if not (away[0] or away[1]):
        return away, None
    dtype, wide = x.dtype, -(-x.shape[1] // 8) * 8
    buffer = torch.empty(((x.shape[0] if away[0] else 0) + (weight.shape[0] if away[1] else 0)) * wide, dtype=dtype,
                         device=x.device)
    to, sets = buffer.data_ptr(), []
    for t, copied in ((x, away[0]), (weight, away[1])):
        if copied:
            rows, cols = t.shape
            sets.append((t.data_ptr(), to, rows, cols, t.stride(0), wide))
            to += rows * wide * _DTYPES[dtype][2]
    call_on(x.device, "gs_rows_pack", (_lib.GsRows * 2)(*sets), len(sets), _DTYPES[dtype][0])
    return away, buffer


def _args(x, weight, buffer, away, bias, residual, out, z, out_dtype, activation) -> _lib.GsLinear:
    (rows, inputs), outputs = x.shape, weight.shape[0]
    code, _, size = _DTYPES[x.dtype]
    if buffer is not None:
        to, wide = buffer.data_ptr(), -(-inputs // 8) * 8
    if away[0]:
        x_at, x_stride = to, wide
        to += rows * wide * size
    else:
        x_at, x_stride = x.data_ptr(), x.stride(0) if rows else 0
    w_at, w_stride = (to, wide) if away[1] else (weight.data_ptr(), weight.stride(0))
    return _lib.GsLinear(x_at, w_at, None if bias is None else bias.data_ptr(),
                         None if residual is None else residual.data_ptr(), None if out is None else out.data_ptr(),
                         None if z is None else z.data_ptr(), rows, x_stride, w_stride,
                         0 if residual is None else residual.stride(0), inputs, outputs, code, _DTYPES[out_dtype][0],
                         0 if z is None else _DTYPES[z.dtype][0], 0 if bias is None else _DTYPES[bias.dtype][0], activation)


def _empty(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _workspace(name: str, a, device):
    n = _lib.size_call(name, C.byref(a))
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


def _forward(x, weight, bias, residual, activation, out_dtype, keep: bool):
    few = x.shape[0] <= FEW_ROWS
    away, buffer = _pack(x, weight, few)
    out = torch.empty((x.shape[0], weight.shape[0]), dtype=out_dtype, device=x.device)
    z = None
    if keep and activation:  # float32 where a bias' gradient sums its slopes; the products round them anyway
        z = torch.empty(out.shape, dtype=x.dtype if bias is None else torch.float32, device=x.device)
    a = _args(x, weight, buffer, away, bias, residual, out, z, out_dtype, activation)
    ws, n = _workspace("gs_linear_fwd_workspace_size", a, x.device)
    call_on(x.device, "gs_linear_fwd", C.byref(a), ptr(ws), n)
    return out, z, buffer, away


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, out_dtype):
        out, z, buffer, away = _forward(x, weight, bias, residual, activation, out_dtype, any(ctx.needs_input_grad[:3]))
        again = x.shape[0] <= FEW_ROWS or _overlaps(x) or _overlaps(weight)  # the backward reads them in other ways
        ctx.save_for_backward(x, weight, bias, z, None if again else buffer)
        ctx.rule, ctx.away = (out_dtype, activation), None if again else away
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        x, weight, bias, z, buffer = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = (None, None, None)
        if need[0] or need[1] or need[2]:
            away = ctx.away
            if away is None:
                away, buffer = _pack(x, weight, False, apart=True)
            d = d_out.contiguous()
            if d.data_ptr() % 16:
                d = d.clone()
            grads = (_empty(x) if need[0] else None, _empty(weight) if need[1] else None, _empty(bias) if need[2] else None)
            a = _args(x, weight, buffer, away, bias, None, None, z, *ctx.rule)
            ws, n = _workspace("gs_linear_bwd_workspace_size", a, x.device)
            call_on(x.device, "gs_linear_bwd", C.byref(a), ptr(d), ptr(grads[0]), ptr(grads[1]), ptr(grads[2]), ptr(ws), n)
        return (*grads, d_out if need[3] else None, None, None)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, [T, N], of x [T, K] and weight [N, K] (one dtype, bfloat16 or float32), bias [N]
    (either) and residual [T, N] (x's dtype, or float32); differentiable in all of them. activation: "none", "relu",
    "gelu" (z Phi(z)), "gelu_tanh" or "silu". The result has the residual's dtype, without one x's. Products and
    epilogue are float32 and rounded once; in the backward pass the output's gradient times act' is rounded to
    x's dtype as an operand of the products (not in the bias' gradient), and act' is taken at z = x weight^T + bias, which the forward
    keeps: in float32, or without a bias in x's dtype. In bfloat16 the activations are off by up to 2^-17 of themselves, in a
    float32 result too. No forward-mode derivative.

    x and weight are read through their row strides where these, the addresses and K are multiples of 16 bytes, and in a
    forward of up to 16 rows wherever the last dimension is contiguous; otherwise they are copied first, at every call, and so are
    rows that overlap (an expanded tensor's) for the backward. Kept for the backward are x, weight, z and, where more than 16 rows
    had to be copied, the copies. T up to 2^28; T N, T K and N K up to 2^33.

    Against the library's product with torch's bias, activation and residual after it this is faster in calls of few rows or few
    tiles and where the epilogue counts (2048 x 1024 -> 4096 with gelu 26 us for 32, 181 x 1024 -> 1024 onto a float32 residual 9 for 47),
    alike in training at 8203 x 1024 -> 4096 and slower in large bare products (8192 x 8192 x 8192 844 us for 679, 16384 x 8192
    -> 2048 506 for 376) and in 16 rows of a large weight (8192 x 8192 32 for 23)."""
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError(f"x must be [tokens, inputs] and weight [outputs, inputs], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise ValueError(f"x and weight must share a dtype, float32 or bfloat16: got {x.dtype}, {weight.dtype}")
    device = x.device
    if not x.is_cuda or weight.device != device:
        raise ValueError("x and weight must be on one GPU")
    n = weight.shape[0]
    if not (1 <= x.shape[1] <= MAX_WIDTH and 1 <= n <= MAX_WIDTH):
        raise ValueError(f"{x.shape[1]} inputs and {n} outputs: 1 to {MAX_WIDTH} are provided")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype not in _DTYPES or bias.device != device:
            raise ValueError(f"bias must be [{n}], float32 or bfloat16, on x's device")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    out_dtype = x.dtype
    if residual is not None:
        if residual.shape != (x.shape[0], n) or residual.device != device or residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"residual must be [{x.shape[0]}, {n}], float32 or x's dtype, on x's device")
        out_dtype, residual = residual.dtype, _rows(residual)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
    x, weight = _rows(x), _rows(weight)
    rest = (bias, residual, ACTIVATIONS[activation], out_dtype)
    if tracked(x, weight, bias, residual):
        return _Linear.apply(x, weight, *rest)
    return _forward(x, weight, *rest, False)[0]
