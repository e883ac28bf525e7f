"""Rotary positions with several axes on the GPU (gs_rotary_axes).

`rotary_axes(q, k, positions, sections)` turns the pairs of every query and key head by angles that
follow the token's place along each axis, e.g. view, row and column of an image patch: the first
sections[0] pairs by axis 0, the next by axis 1, and so on. Queries and keys go in one launch, read
through their strides (slices of a packed projection), the angles formed once per token. The
gradient is the same turn backwards.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._grad import tracked
from ._lib import call

MAX_AXES, MAX_PAIRS = 4, 256  # GS_ROTARY_MAX_AXES, GS_ROTARY_MAX_PAIRS
_DTYPES = {torch.float32: _lib.GS_FLOAT32, torch.bfloat16: _lib.GS_BFLOAT16}
_FLAGS = {"half": 0, "adjacent": _lib.GS_ROTARY_ADJACENT, "axis": 0, "shared": _lib.GS_ROTARY_SHARED}


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _turn(q, k, positions, sections, base: float, flags: int):
    q = _rows(q)
    tokens, heads, dim = q.shape
    q_out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    q_token, q_head, _ = q.stride()
    k_out, k_at, k_to, k_token, k_head, k_heads = None, None, None, 0, 0, 0
    if k is not None:
        k = _rows(k)
        k_heads = k.shape[1]
        k_out = torch.empty((tokens, k_heads, dim), dtype=q.dtype, device=q.device)
        k_at, k_to = k.data_ptr(), k_out.data_ptr()
        k_token, k_head, _ = k.stride()
    a = _lib.GsRotary(q.data_ptr(), k_at, q_out.data_ptr(), k_to, positions.data_ptr(), tokens, q_token, q_head, k_token,
                      k_head, base, heads, k_heads, dim, len(sections), sections, _DTYPES[q.dtype], flags)
    call("gs_rotary_axes", C.byref(a), _lib.stream_handle(q.device))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base, flags):
        ctx.save_for_backward(positions)
        ctx.rule = (sections, base, flags ^ _lib.GS_ROTARY_INVERSE)
        return _turn(q, k, positions, sections, base, flags)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_q, d_k):
        (positions,) = ctx.saved_tensors
        d_q, d_k = _turn(d_q, d_k, positions, *ctx.rule)
        return d_q, d_k, None, None, None, None


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, sections, *,
                base: float = 10000.0, pairing: str = "half", spectrum: str = "axis"):
    """(q', k') for q [T, heads, D] and k [T, kv_heads, D] (k None: q' alone), bfloat16 or float32,
    differentiable in q and k. positions [T, axes]: float32 (or integers), one coordinate per axis.
    sections: the number of pairs of each axis, P in all, 2 P <= D; elements from 2 P on are copied.

    pairing "half": pair p is the elements (p, p + P); "adjacent": (2 p, 2 p + 1). The angle is
    position * base^-x: spectrum "axis" runs x over [0, 1) within each section, "shared" over all
    P pairs. The angle is formed to float32's last place for positions up to 2^30 (2^28
    turns). Integer positions are taken as float32, which holds them exactly up to 2^24."""
    if q.dim() != 3 or (k is not None and k.dim() != 3):
        raise ValueError("q and k must be [tokens, heads, D]")
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
        raise ValueError("q and k must share a dtype, float32 or bfloat16")
    if not q.is_cuda or (k is not None and k.device != q.device) or positions.device != q.device:
        raise ValueError("q, k and positions must be on one GPU")
    if k is not None and (k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}")
    if q.shape[1] < 1 or (k is not None and k.shape[1] < 1):
        raise ValueError("need at least one head")
    sections = tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections: 1 to {MAX_AXES} pair counts")
    pairs = sum(sections)
    if not 1 <= pairs <= MAX_PAIRS or 2 * pairs > q.shape[2]:
        raise ValueError(f"{pairs} pairs do not fit heads of {q.shape[2]} elements (at most {MAX_PAIRS} pairs)")
    if positions.dim() != 2 or positions.shape != (q.shape[0], len(sections)):
        raise ValueError(f"positions must be [{q.shape[0]}, {len(sections)}], got {tuple(positions.shape)}")
    if positions.dtype not in (torch.float32, torch.int32, torch.int64, torch.int16):
        raise ValueError("positions must be float32 or integers")
    if pairing not in ("half", "adjacent"):
        raise ValueError('pairing must be "half" or "adjacent"')
    if spectrum not in ("axis", "shared"):
        raise ValueError('spectrum must be "axis" or "shared"')
    base = float(base)
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError("base must be positive and finite")
    positions = positions.detach()
    if positions.dtype != torch.float32 or not positions.is_contiguous():
        positions = positions.to(torch.float32).contiguous()
    flags = _FLAGS[pairing] | _FLAGS[spectrum]
    if tracked(q, k):
        q2, k2 = _Rotary.apply(q, k, positions, sections, base, flags)
    else:
        q2, k2 = _turn(q, k, positions, sections, base, flags)
    return q2 if k is None else (q2, k2)
