"""A gated linear recurrence over packed documents on the GPU (gs_gated_scan_fwd / gs_gated_scan_bwd).

`gated_scan(x, forget, gate)` mixes the tokens of a scene in order, in time and memory linear in their number,
where `attention` goes by the square: a predictor on long captures runs it in some of its layers. A scene
that grows keeps one row of state instead of a cache.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._grad import tracked
from ._lib import call_on, ptr

MAX_WIDTH, MAX_DOCS = 1 << 20, (1 << 30) - 1  # GS_SCAN_MAX_WIDTH, and what gs_gated_scan_fwd takes
_DTYPES = {torch.float32: _lib.GS_FLOAT32, torch.bfloat16: _lib.GS_BFLOAT16}


def _rows(t):
    return t if t is None or ((t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0) else t.contiguous()


def _args(x, forget, gate, initial, offsets, reverse, y, state, carry) -> _lib.GsGatedScan:
    return _lib.GsGatedScan(x.data_ptr(), forget.data_ptr(), None if gate is None else gate.data_ptr(),
                            None if initial is None else initial.data_ptr(), ptr(y), ptr(state), ptr(carry),
                            None if offsets is None else offsets.data_ptr(), x.shape[0], x.stride(0), forget.stride(0),
                            0 if gate is None else gate.stride(0), 1 if offsets is None else offsets.shape[0] - 1,
                            x.shape[1], _DTYPES[x.dtype], reverse)


def _workspace(x):
    n = _lib.size_call("gs_gated_scan_workspace_size", x.shape[0], x.shape[1])
    return (torch.empty(n, dtype=torch.uint8, device=x.device), n) if n else (None, 0)


def _forward(x, forget, gate, initial, offsets, reverse, keep: bool, want_state: bool):
    docs = 1 if offsets is None else offsets.shape[0] - 1
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    state = torch.empty((docs, x.shape[1]), dtype=torch.float32, device=x.device) if want_state else None
    carry = None
    if keep:
        chunks = _lib.size_call("gs_gated_scan_chunks", x.shape[0])
        carry = torch.empty((chunks, x.shape[1]), dtype=torch.float32, device=x.device)
    a = _args(x, forget, gate, initial, offsets, reverse, y, state, carry)
    ws, n = _workspace(x)
    call_on(x.device, "gs_gated_scan_fwd", C.byref(a), ptr(ws), n)
    return y, state, carry


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, forget, gate, initial, offsets, reverse, want_state):
        y, state, carry = _forward(x, forget, gate, initial, offsets, reverse, True, want_state)
        ctx.save_for_backward(x, forget, gate, initial, offsets, carry)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_state):
        if d_y is None and d_state is None:
            return (None,) * 7
        x, forget, gate, initial, offsets, carry = ctx.saved_tensors
        d_y = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if d_y is None else d_y.contiguous()
        d_state = None if d_state is None else d_state.contiguous()
        outs = [torch.empty(t.shape, dtype=t.dtype, device=x.device) if t is not None and need else None
                for t, need in zip((x, forget, gate, initial), ctx.needs_input_grad)]
        a = _args(x, forget, gate, initial, offsets, ctx.reverse, None, None, carry)
        ws, n = _workspace(x)
        call_on(x.device, "gs_gated_scan_bwd", C.byref(a), ptr(d_y), ptr(d_state), *map(ptr, outs), ptr(ws), n)
        return (*outs, None, None, None)


def gated_scan(x: torch.Tensor, forget: torch.Tensor, gate: torch.Tensor | None = None, *,
               offsets: torch.Tensor | None = None, initial: torch.Tensor | None = None, reverse: bool = False,
               return_state: bool = False):
    """y [T, C] (and with return_state the states [docs, C], float32) of the recurrence

        h_t = a_t h_(t-1) + (1 - a_t) x_t,  a = sigmoid(forget),     y_t = h_t, or with gate: h_t silu(gate_t)

    over each document's tokens in order (reverse: from its last to its first), from h = initial [docs, C] (float32;
    None: zero). x, forget and gate are [T, C] of one dtype, bfloat16 or float32. offsets [docs + 1] int32,
    non-decreasing: document d's tokens are offsets[d] .. offsets[d + 1] (None: one document of all tokens); tokens
    outside all documents give 0. A state is h after the document's last step, an empty document's its initial
    one: given back as `initial`, the next tokens continue where these ended. Differentiable in x, forget, gate
    and initial, through y and the states. h is float32; the smaller of a and 1 - a is off by 2^-23 |forget| of itself (the
    hardware's exponential, in float32 too). Documents do not reach each other, whatever they hold; differences
    x - h have to be finite in float32. C up to 2^20, T times C / 256 (rounded up) up to 2^29, docs below
    2^30. No forward-mode derivative."""
    if x.dim() != 2:
        raise ValueError("x must be [tokens, width]")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError("x must be on the GPU")
    for t, name in ((forget, "forget"), (gate, "gate")):
        if t is None and name == "gate":
            continue
        if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"{name} must have x's shape, dtype and device")
    if not 1 <= x.shape[1] <= MAX_WIDTH:
        raise ValueError(f"width {x.shape[1]}: 1 to {MAX_WIDTH} are provided")
    docs = 1
    if offsets is not None:
        if not (isinstance(offsets, torch.Tensor) and offsets.dtype == torch.int32 and offsets.dim() == 1
                and offsets.is_contiguous() and offsets.device == x.device and offsets.shape[0] >= 2):
            raise ValueError("offsets must be a contiguous int32 tensor of at least 2 entries on x's device")
        docs = offsets.shape[0] - 1
        if docs > MAX_DOCS:
            raise ValueError(f"{docs} documents: up to {MAX_DOCS} are provided")
    if initial is not None:
        if initial.shape != (docs, x.shape[1]) or initial.dtype != torch.float32 or initial.device != x.device:
            raise ValueError(f"initial must be float32 [{docs}, {x.shape[1]}] on x's device")
        initial = initial if initial.is_contiguous() else initial.contiguous()
    args = (_rows(x), _rows(forget), _rows(gate), initial, offsets, bool(reverse))
    if tracked(x, forget, gate, initial):
        y, state = _GatedScan.apply(*args, bool(return_state))
    else:
        y, state, _ = _forward(*args, False, bool(return_state))
    return (y, state) if return_state else y
