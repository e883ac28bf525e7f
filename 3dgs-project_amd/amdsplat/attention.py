"""Softmax attention over packed documents on the GPU (gs_attention_fwd / gs_attention_bwd).

`attention(q, k, v, ...)` is what a splat predictor (a transformer over the tokens of posed views
whose output is a set of Gaussians) runs between its projections. The tokens of several scenes are
packed one after the other; a scene is a document and sees itself only. Query heads may share key
heads; scores may be capped by a tanh; the causal mask may leave a prefix that all tokens see; keys
and values may be a cache that is longer than what it holds. bfloat16 or float32 CUDA tensors;
statistics and sums are float32. Nothing is read back to the host.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._grad import tracked
from ._lib import call, ptr

MAX_DIM = 128  # GS_ATTENTION_MAX_DIM
_DTYPES = {torch.float32: (_lib.GS_FLOAT32, 4), torch.bfloat16: (_lib.GS_BFLOAT16, 8)}


def _readable(t: torch.Tensor, group: int = 0) -> torch.Tensor:
    """t itself if the kernels can read it through its strides, otherwise a contiguous copy. group: query
    heads to a key head (q: 64 consecutive rows have to span less than 2^28 elements)."""
    per = _DTYPES[t.dtype][1]
    st, sh, sd = t.stride()
    if 0 in t.shape:
        return t
    ok = ((sd == 1 or t.shape[2] == 1) and 0 <= st < 1 << 22 and 0 <= sh < 1 << 40 and st % per == 0 and sh % per == 0
          and t.data_ptr() % 16 == 0 and (not group or (64 // group + 2) * st + group * sh < 1 << 28))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _at(t) -> int | None:
    return None if t is None else t.data_ptr()


def _args(q, k, v, out, low, lse, offsets, k_offsets, k_lengths, prefix, causal, softcap, scale) -> _lib.GsAttention:
    tq, heads, dim = q.shape
    tk, kv_heads, _ = k.shape
    q_token, q_head, _ = q.stride() if tq else (0, 0, 1)
    (k_token, k_head, _), (v_token, v_head, _) = (k.stride(), v.stride()) if tk else ((0, 0, 1), (0, 0, 1))
    return _lib.GsAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _at(low), lse.data_ptr(),
                            _at(offsets), _at(k_offsets), _at(k_lengths), _at(prefix), tq, tk, q_token, q_head,
                            k_token, k_head, v_token, v_head, 1 if offsets is None else offsets.shape[0] - 1, heads,
                            kv_heads, dim, _DTYPES[q.dtype][0], causal, softcap, scale)


def _workspace(name: str, args, device):
    n = _lib.size_call(name, C.byref(args))
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


def _forward(q, k, v, offsets, k_offsets, k_lengths, prefix, causal, softcap, scale, low=None):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    args = _args(q, k, v, out, low, lse, offsets, k_offsets, k_lengths, prefix, causal, softcap, scale)
    ws, n = _workspace("gs_attention_fwd_workspace_size", args, q.device)
    call("gs_attention_fwd", C.byref(args), ptr(ws), n, _lib.stream_handle(q.device))
    return out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, k_offsets, k_lengths, prefix, causal, softcap, scale):
        q, k, v = _readable(q, q.shape[1] // k.shape[1]), _readable(k), _readable(v)
        # what rounding takes off the output, for the gradient's row sums
        low = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q.dtype == torch.bfloat16 else None
        out, lse = _forward(q, k, v, offsets, k_offsets, k_lengths, prefix, causal, softcap, scale, low)
        ctx.save_for_backward(q, k, v, out, low, lse, offsets, k_offsets, k_lengths, prefix)
        ctx.rule = (causal, softcap, scale)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)  # (a zero gradient for lse would be a launch that nothing reads)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, _d_lse):
        if d_out is None:
            return (None,) * 10
        q, k, v, out, low, lse, offsets, k_offsets, k_lengths, prefix = ctx.saved_tensors
        d_out = d_out.contiguous()
        if d_out.numel() and d_out.data_ptr() % 16:
            d_out = d_out.clone()
        d_q, d_k, d_v = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        args = _args(q, k, v, out, low, lse, offsets, k_offsets, k_lengths, prefix, *ctx.rule)
        ws, n = _workspace("gs_attention_bwd_workspace_size", args, q.device)
        call("gs_attention_bwd", C.byref(args), ptr(d_out), ptr(d_q), ptr(d_k), ptr(d_v), ptr(ws), n,
             _lib.stream_handle(q.device))
        return (d_q, d_k, d_v) + (None,) * 7


def _table(t, name: str, n: int, device) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous()
            and t.device == device):
        raise ValueError(f"{name} must be a contiguous int32 tensor on the tensors' device")
    if t.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, got {t.shape[0]}")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, offsets: torch.Tensor | None = None,
              k_offsets: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None, causal: bool = False,
              prefix: torch.Tensor | None = None, softcap: float = 0.0, scale: float | None = None,
              return_lse: bool = False):
    """out [Tq, heads, D] (and with return_lse the float32 log-sum-exp [Tq, heads], which takes no
    gradient) of q [Tq, heads, D] over k, v [Tk, kv_heads, D]; differentiable in q, k and v.

    offsets [docs + 1] int32, non-decreasing: document d's tokens are offsets[d] .. offsets[d + 1]
    (None: one document of all tokens). k_offsets: the same for the keys (None: as the queries).
    k_lengths [docs] int32: of a document's key tokens only the first so many are there (a cache);
    the rest may hold anything. causal: query i of a document of Lq queries and Lk keys sees key j
    if j <= i + Lk - Lq; prefix [docs] int32 (with causal): or if j < prefix[d]. softcap c (0, or 2^-96 to 2^96):
    scores s become c tanh(s / c). scale: of the scores before the cap (default 1 / sqrt(D)).

    A query that sees no key gets 0 and -infinity. A key or value that is not finite reaches only the
    queries that see it (the gradients of its document are not kept apart so). Sums are float32: 2^8
    times the sum of |v| over a query's keys has to be finite there. No forward-mode derivative. D up to
    128 (padded to a multiple of 8 by a copy). Tensors are read through their strides where these and the
    addresses are multiples of 16 bytes and the last dimension is contiguous; otherwise they are copied
    first."""
    if not (q.dim() == k.dim() == v.dim() == 3):
        raise ValueError("q, k and v must be [tokens, heads, D]")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must share a dtype, float32 or bfloat16: got {q.dtype}, {k.dtype}, {v.dtype}")
    device = q.device
    if not q.is_cuda or k.device != device or v.device != device:
        raise ValueError("q, k and v must be on one GPU")
    (tq, heads, d), (tk, kv_heads, _) = q.shape, k.shape
    if k.shape != v.shape or k.shape[2] != d:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not 1 <= d <= MAX_DIM:
        raise ValueError(f"head size {d}: 1 to {MAX_DIM} are provided")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
    if heads // kv_heads > 512:
        raise ValueError("at most 512 heads may share a key head")
    if offsets is None and k_offsets is not None:
        raise ValueError("k_offsets without offsets")
    docs = 1
    if offsets is not None:
        docs = offsets.numel() - 1 if isinstance(offsets, torch.Tensor) else 0
        if docs < 1:
            raise ValueError("offsets must have at least 2 entries")
        _table(offsets, "offsets", docs + 1, device)
        if k_offsets is None:
            if tk != tq:
                raise ValueError(f"{tk} keys for {tq} queries: pass k_offsets")
            k_offsets = offsets
        else:
            _table(k_offsets, "k_offsets", docs + 1, device)
    if k_lengths is not None:
        _table(k_lengths, "k_lengths", docs, device)
    if prefix is not None:
        if not causal:
            raise ValueError("a prefix needs causal=True")
        _table(prefix, "prefix", docs, device)
    softcap = float(softcap)
    if softcap != 0.0 and not 2.0 ** -96 <= softcap <= 2.0 ** 96:
        raise ValueError("softcap must be 0 or between 2^-96 and 2^96")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if scale != 0.0 and not 2.0 ** -126 <= abs(scale) <= 2.0 ** 126:
        raise ValueError("scale must be finite, 0 or between 2^-126 and 2^126 in size")
    if softcap and scale and not 2.0 ** -126 <= abs(scale) / softcap <= 2.0 ** 125:
        raise ValueError("scale / softcap must be between 2^-126 and 2^125")
    if d % 8:
        q, k, v = (torch.nn.functional.pad(t, (0, -d % 8)) for t in (q, k, v))
    rest = (offsets, k_offsets, k_lengths, prefix, bool(causal), softcap, scale)
    if tracked(q, k, v):
        out, lse = _Attention.apply(q, k, v, *rest)
    else:
        out, lse = _forward(_readable(q, heads // kv_heads), _readable(k), _readable(v), *rest)
    if d % 8:
        out = out[..., :d]
    return (out, lse) if return_lse else out
