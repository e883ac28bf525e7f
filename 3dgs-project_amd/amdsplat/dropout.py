"""Dropout whose mask is never stored (gs_dropout): every element's bits come from a counter-based generator, so the
backward pass, or a replayed graph, forms them again from the seed.
"""
from __future__ import annotations

import torch

from . import _lib
from ._grad import tracked
from ._lib import call_on

_DTYPES = {torch.float32: _lib.GS_FLOAT32, torch.bfloat16: _lib.GS_BFLOAT16}


def check_rule(p, seed, draw, device):
    """(p, device seed or None, host seed, draw) of an operator's arguments."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError("the dropout probability must be at least 0 and below 1")
    draw = int(draw)
    if not 0 <= draw < 1 << 64:
        raise ValueError("draw must be between 0 and 2^64 - 1")
    if p == 0.0:
        return 0.0, None, 0, draw
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError("seed must be an integer, or an int64 tensor of one element on the tensors' device")
        return p, seed, 0, draw
    if seed is None or isinstance(seed, bool) or not isinstance(seed, int):
        raise ValueError("dropout needs a seed: an integer, or an int64 tensor of one element on the tensors' device")
    if not -(1 << 63) <= seed < 1 << 64:
        raise ValueError("seed must have 64 bits")
    return p, None, seed % (1 << 64), draw


def _drop(x, rule):
    p, seed_at, seed, draw = rule
    width = x.shape[-1] if x.dim() else 1
    rows = x.numel() // width if width else 0
    if x.dim() == 2 and (x.stride(1) == 1 or width == 1) and x.stride(0) >= 0:
        stride = x.stride(0)
    else:
        x, stride = x.contiguous(), width
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    call_on(x.device, "gs_dropout", x.data_ptr(), out.data_ptr(), rows, stride, width, _DTYPES[x.dtype], p,
            None if seed_at is None else seed_at.data_ptr(), seed, draw)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed_at, seed, draw):
        ctx.save_for_backward(seed_at)
        ctx.rule = (p, seed, draw)
        return _drop(x, (p, seed_at, seed, draw))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        (seed_at,) = ctx.saved_tensors
        p, seed, draw = ctx.rule
        return _drop(d_out, (p, seed_at, seed, draw)), None, None, None, None


def dropout(x: torch.Tensor, p: float, seed, *, draw: int = 0) -> torch.Tensor:
    """x with elements dropped with probability p (0 <= p < 1, taken as a multiple of 2^-16) and the others
    divided by 1 - p; bfloat16 or float32 on the GPU, differentiable in x. Every dimension but the last, which is
    below 2^31, counts as rows; rows times an eighth of it (rounded up) stay below 2^32 - 256.

    seed: an integer, or an int64 CUDA tensor of one element, read when the kernels run (so a captured graph
    may be replayed with another seed; the backward pass reads it again, and autograd refuses one that was written
    in between). draw: which dropout of a step this is; masks of different seeds or draws are independent,
    the same seed, draw and shape give the same mask. The generator is Philox4x32-10, 16 bits an element, key = seed,
    counter = (column / 8, row, draw). What is dropped is 0 whatever it was. No forward-mode derivative."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError("x must be on the GPU")
    rule = check_rule(p, seed, draw, x.device)
    if x.dim() and x.shape[-1] >= 1 << 31:
        raise ValueError("the last dimension must be below 2^31")
    if x.dim() and x.numel() // max(x.shape[-1], 1) >= 1 << 32:
        raise ValueError("at most 2^32 - 1 rows")
    return _Dropout.apply(x, *rule) if tracked(x) else _drop(x, rule)
