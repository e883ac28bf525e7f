"""The global gradient norm over many tensors and clipping by it (gs_grad_norm, gs_grad_scale).

`grad_norm(grads)` and `clip_grad_norm(grads, max_norm)` take any number of float32 and bfloat16
gradients in a few launches; the norm is summed in float64 in a fixed order and stays on the device
(no host synchronisation). `FusedAdam.step(max_norm=...)` clips inside the update instead, without a
pass over the gradients of its own.
"""
from __future__ import annotations

from array import array

import torch

from . import _lib
from ._grad import refuse_tangents
from ._lib import call

_DTYPES = {torch.float32: _lib.GS_FLOAT32, torch.bfloat16: _lib.GS_BFLOAT16}


class _Tensors:
    """The host tables of a call. `keep` holds what they point to."""

    def __init__(self, grads, what: str):
        self.keep = grads
        try:
            self.dtypes = array("i", [_DTYPES[t.dtype] for t in grads])
        except KeyError:
            raise ValueError(f"{what} must be float32 or bfloat16") from None
        self.device = grads[0].device
        dev = self.device
        if dev.type != "cuda" or any(t.device != dev for t in grads):
            raise ValueError(f"{what} must be on one GPU")
        self.sizes = array("q", [t.numel() for t in grads])
        self.ptrs = array("Q", [t.data_ptr() for t in grads])
        self.n = len(grads)


def _at(a: array) -> int:
    return a.buffer_info()[0]


def _list(grads, what: str):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        raise ValueError(f"{what}: no tensors")
    if any(not isinstance(t, torch.Tensor) or t.layout != torch.strided for t in grads):
        raise ValueError(f"{what} must be dense tensors")
    refuse_tangents(grads, what)
    return grads


def _norm(t: _Tensors, max_norm):
    out = torch.empty(2, dtype=torch.float32, device=t.device)
    n = _lib.size_call("gs_grad_norm_workspace_size", _at(t.sizes), t.n)
    ws = torch.empty(max(n, 8), dtype=torch.uint8, device=t.device)
    call("gs_grad_norm", _at(t.ptrs), _at(t.sizes), _at(t.dtypes), t.n, 0.0 if max_norm is None else max_norm,
         out.data_ptr(), None if max_norm is None else out.data_ptr() + 4, ws.data_ptr(), n,
         _lib.stream_handle(t.device))
    return out[0], out[1]


def check_max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be >= 0")
    return max_norm


@torch.no_grad()
def grad_norm(grads) -> torch.Tensor:
    """sqrt of the sum of all squares of a tensor or an iterable of tensors: a 0-dim float32 device
    tensor. Non-contiguous tensors are copied."""
    grads = [t if t.is_contiguous() else t.contiguous() for t in _list(grads, "gradients")]
    return _norm(_Tensors(grads, "gradients"), None)[0]


@torch.no_grad()
def clip_grad_norm(grads, max_norm: float, out=None) -> torch.Tensor:
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)), in place or into the tensors `out`
    (of the gradients' shapes or flat, of their dtypes, not overlapping them), and returns the norm before clipping (a
    0-dim float32 device tensor). A norm that is infinite or NaN leaves no gradient usable, as the
    product says; the caller checks the returned norm."""
    grads = _list(grads, "gradients")
    max_norm = check_max_norm(max_norm)
    if any(not t.is_contiguous() for t in grads):
        raise ValueError("gradients must be contiguous")
    t = _Tensors(grads, "gradients")
    to = t
    if out is not None:
        out = _list(out, "out")
        if len(out) != t.n:
            raise ValueError(f"{len(out)} outputs for {t.n} gradients")
        if any(not o.is_contiguous() for o in out):
            raise ValueError("out must be contiguous")
        to = _Tensors(out, "out")
        if (any(o.shape != g.shape and (o.dim() != 1 or o.numel() != g.numel()) for o, g in zip(out, grads))
                or to.dtypes != t.dtypes or to.device != t.device):
            raise ValueError("out must have the gradients' shapes (or be flat) and dtypes, on their device")
    norm, coef = _norm(t, max_norm)
    call("gs_grad_scale", _at(t.ptrs), _at(to.ptrs), _at(t.sizes), _at(t.dtypes), t.n, coef.data_ptr(),
         _lib.stream_handle(t.device))
    torch.autograd.graph.increment_version(to.keep)  # autograd sees the writes
    return norm


def clip_coefficient(grads, max_norm):
    """(norm, min(1, max_norm / (norm + 1e-6))) as 0-dim float32 device tensors."""
    return _norm(_Tensors(_list(grads, "gradients"), "gradients"), check_max_norm(max_norm))
