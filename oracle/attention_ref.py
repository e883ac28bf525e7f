"""Packed attention with its gradients in float64 on the CPU, written from the formulas, and for
each output an elementwise bound on what a kernel may be off.

The bounds follow the kernels' roundings. u is the type's unit roundoff (2^-8 bfloat16, 2^-24
float32); the inputs are exact. Scores are float32 dot products of D terms and probabilities follow
them through an exponential, so a probability's relative error is at most
    e_i = 2^-23 ((D + 4) max_j scale sum_d |q_d k_d| + Lk + 16) + 2^-20 cap,
the last for the capped scores' tanh (float32's own is better). Probabilities and their gradients
are rounded once to the type (u), sums are float32 (in e), outputs are rounded once (u):
    |d out|  <= (2u + 2e) sum_j p |v|
    |d D_i|  <= sum_d |dO| (2u + 2e) sum_j p |v| + e sum_d |dO| |o|            (D_i = dO . o)
    |d ds|   <= u |ds| + slope p |d D| + 3 e p (|dO||v| + |D|)
    |d dq|   <= scale sum_j |d ds| |k| + u |dq|,   dk and dv likewise.
A probability below float32's smallest normal number is zero: 1e-30 in the place of 0.
"""
import math

import torch

F64 = torch.float64
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def visible(nq, nk, causal, prefix):
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
    see = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        see = (j <= i + nk - nq) | (j < prefix)
    return see


def forward64(q, k, v, see, scale, cap):
    """out, lse, p, slope of one head, in float64; rows that see nothing give 0 and -inf."""
    s = scale * (q @ k.t())
    slope = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s, slope = cap * t, 1 - t * t
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    live = see.any(1)
    p = torch.zeros_like(s)
    p[live] = torch.softmax(s[live], 1)
    lse = torch.full((q.shape[0],), -math.inf, dtype=F64)
    lse[live] = torch.logsumexp(s[live], 1)
    return p @ v, lse, p, slope


def attention(q, k, v, q_at, k_at, k_len=None, causal=False, prefix=None, softcap=0.0, scale=None, d_out=None):
    """q [Tq, H, D], k, v [Tk, Hk, D] on the CPU in the kernel's dtype; q_at, k_at: document offsets.
    Returns {name: (value, bound)} for out, lse and, with d_out, d_q, d_k, d_v."""
    u = UNIT[q.dtype]
    heads, kv_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    names = ["out", "lse"] + (["d_q", "d_k", "d_v"] if d_out is not None else [])
    like = dict(out=q, lse=q[..., 0], d_q=q, d_k=k, d_v=v)
    r = {n: [torch.zeros_like(like[n]), torch.zeros_like(like[n])] for n in names}
    r["lse"][0].fill_(-math.inf)
    for d in range(len(q_at) - 1):
        rows = slice(q_at[d], q_at[d + 1])
        nq = q_at[d + 1] - q_at[d]
        nk = k_at[d + 1] - k_at[d] if k_len is None else k_len[d]
        keys = slice(k_at[d], k_at[d] + nk)
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, causal, 0 if prefix is None else prefix[d])
        for h in range(heads):
            g = h // (heads // kv_heads)
            a, b, w = q[rows, h], k[keys, g], v[keys, g]
            o, lse, p, slope = forward64(a, b, w, see, scale, softcap)
            size = abs(scale) * (a.abs() @ b.abs().t())
            e = 2.0 ** -23 * ((dim + 4) * size.amax(1) + nk + 16) + 2.0 ** -20 * softcap
            e = e[:, None]
            r["out"][0][rows, h], r["lse"][0][rows, h] = o, lse
            away = (2 * u + 2 * e) * (p @ w.abs())
            r["out"][1][rows, h] = away + 1e-30
            r["lse"][1][rows, h] = e[:, 0] + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)
            if d_out is None:
                continue
            go = d_out[rows, h].to(F64)
            delta = (go * o).sum(1, keepdim=True)
            dp = go @ w.t()
            ds = p * (dp - delta) * slope
            off_delta = (go.abs() * away).sum(1, keepdim=True) + e * (go.abs() * o.abs()).sum(1, keepdim=True)
            off = u * ds.abs() + slope * p * off_delta + 3 * e * p * (go.abs() @ w.abs().t() + delta.abs())
            off = off * (1 + 2 * u) + 1e-30 * see
            dq, dk, dv = scale * (ds @ b), scale * (ds.t() @ a), p.t() @ go
            r["d_q"][0][rows, h] = dq
            r["d_q"][1][rows, h] = abs(scale) * (off @ b.abs()) + u * dq.abs()
            r["d_k"][0][keys, g] += dk
            r["d_k"][1][keys, g] += abs(scale) * (off.t() @ a.abs()) + (u + 2.0 ** -22) * abs(scale) * (ds.abs().t() @ a.abs())
            r["d_v"][0][keys, g] += dv
            r["d_v"][1][keys, g] += (2 * u * p + 2 * e * p + 1e-30 * see).t() @ go.abs()
    return {n: tuple(x) for n, x in r.items()}
