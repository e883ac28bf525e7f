"""The operators of a predictor's block in float64, from their definitions: projections with an epilogue, norms around a
residual branch, dropout's bits, the gated recurrence. Every function gives (values, sizes): dicts of tensors where a
size is the value's formula with each term replaced by its absolute value, which is what a float32
evaluation's rounding is relative to.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def wide(t):
    return None if t is None else t.detach().double()


# ---- dropout -----------------------------------------------------------------------------------------


def philox(counter, key):
    """Philox4x32-10 of one counter of four words under a key of two, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def keep(rows, width, seed, draw, p):
    """The factors [rows, width]: 0 or 2^16 / (2^16 - t), t = round(2^16 p)."""
    t = min(int(math.floor(p * 65536 + 0.5)), 65535)
    groups = -(-width // 8)
    u = np.uint64
    low, half = u(0xffffffff), u(32)
    x = [np.tile(np.arange(groups, dtype=u), rows), np.repeat(np.arange(rows, dtype=u), groups)]
    x += [np.full_like(x[0], draw & 0xffffffff), np.full_like(x[0], draw >> 32)]
    k = [seed & 0xffffffff, seed >> 32 & 0xffffffff]
    for _ in range(10):
        a, b = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [b >> half ^ x[1] ^ u(k[0]), b & low, a >> half ^ x[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    bits = np.stack([h for w in x for h in (w & u(0xffff), w >> u(16))], -1).reshape(rows, groups * 8)[:, :width]
    return torch.from_numpy((bits >= u(t)) * (65536.0 / (65536 - t)))


# ---- norms -------------------------------------------------------------------------------------------


def _standard(v, size, layer, eps):
    """(v^, 1 / deviation, size of v^)."""
    mean = v.mean(1, keepdim=True) if layer else 0.0
    c = v - mean
    inv = (c.square().mean(1, keepdim=True) + eps) ** -0.5
    return c * inv, inv, (size + (size.mean(1, keepdim=True) if layer else 0.0)) * inv


def _standard_gradient(d, d_size, hat, inv, hat_size, layer):
    m = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    value = d - hat * m(d * hat) - (m(d) if layer else 0.0)
    return value * inv, (d_size + hat_size * m(d_size * hat_size) + (m(d_size) if layer else 0.0)) * inv


def residual_norm(x, y, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, *, kind="rms", eps=1e-6,
                  scale=1.0, factors=None, d_h=None, d_n=None):
    """y None: the norm of x alone. factors: dropout's, or None."""
    layer = kind == "layer"
    x, y, weight, bias, post_weight, post_bias, gate = map(wide, (x, y, weight, bias, post_weight, post_bias, gate))
    one = torch.ones((), dtype=torch.float64, device=x.device)
    w, g, k = (one if t is None else t for t in (weight, gate, factors))
    h, h_size = x, x.abs()
    if y is not None:
        b, b_size = y, y.abs()
        if post_weight is not None:
            y_hat, y_inv, y_size = _standard(y, y.abs(), layer, eps)
            shift = 0.0 if post_bias is None else post_bias
            b, b_size = y_hat * post_weight + shift, y_size * post_weight.abs() + abs(shift)
        u, u_size = b * k, b_size * k
        h, h_size = x + scale * g * u, x.abs() + abs(scale) * g.abs() * u_size
    hat, inv, hat_size = _standard(h, h_size, layer, eps)
    n, n_size = hat * w, hat_size * w.abs()
    if bias is not None:
        n, n_size = n + bias, n_size + bias.abs()
    value, size = {"h": h, "n": n}, {"h": h_size, "n": n_size}
    if d_h is None and d_n is None:
        return value, size
    d_h, d_n = (torch.zeros_like(x) if t is None else wide(t) for t in (d_h, d_n))
    d, d_size = _standard_gradient(d_n * w, (d_n * w).abs(), hat, inv, hat_size, layer)
    d, d_size = d + d_h, d_size + d_h.abs()

    def put(name, v, s):
        value[name], size[name] = v, s

    put("d_x", d, d_size)
    put("d_weight", (d_n * hat).sum(0), (d_n.abs() * hat_size).sum(0))
    put("d_bias", d_n.sum(0), d_n.abs().sum(0))
    if y is None:
        return value, size
    e, e_size = scale * d * u, abs(scale) * d_size * u_size
    put("d_gate", e, e_size)
    if gate is not None and gate.dim() == 1:
        put("d_gate", e.sum(0), e_size.sum(0))
    v, v_size = scale * d * g * k, abs(scale) * d_size * g.abs() * k
    if post_weight is not None:
        put("d_post_weight", (v * y_hat).sum(0), (v_size * y_size).sum(0))
        put("d_post_bias", v.sum(0), v_size.sum(0))
        v, v_size = _standard_gradient(v * post_weight, v_size * post_weight.abs(), y_hat, y_inv, y_size, layer)
    put("d_y", v, v_size)
    return value, size


# ---- the recurrence ----------------------------------------------------------------------------------


def gated_scan(x, forget, gate=None, *, offsets=None, initial=None, reverse=False, d_y=None, d_state=None):
    """Token by token. offsets: a list, or None for one document."""
    tokens, width = x.shape
    offsets = [0, tokens] if offsets is None else offsets
    docs = len(offsets) - 1
    x, f, o, initial, d_y, d_state = map(wide, (x, forget, gate, initial, d_y, d_state))
    zero = torch.zeros(docs, width, dtype=torch.float64, device=x.device)
    a, rest = torch.sigmoid(f), torch.sigmoid(-f)
    p = torch.ones_like(x) if o is None else torch.sigmoid(o)
    open_ = p if o is None else o * p
    state, state_size = (zero.clone() if initial is None else initial.clone() for _ in range(2))
    state_size = state_size.abs()
    before, before_size, after, after_size = (torch.zeros_like(x) for _ in range(4))
    order = [range(offsets[d], offsets[d + 1]) for d in range(docs)]
    if reverse:
        order = [r[::-1] for r in order]
    for d, rows in enumerate(order):
        for t in rows:
            before[t], before_size[t] = state[d], state_size[d]
            state[d] = a[t] * state[d] + rest[t] * x[t]
            state_size[d] = a[t] * state_size[d] + rest[t] * x[t].abs()
            after[t], after_size[t] = state[d], state_size[d]
    value, size = {"y": after * open_, "state": state}, {"y": after_size * open_.abs(), "state": state_size}
    if d_y is None and d_state is None:
        return value, size
    d_y = torch.zeros_like(x) if d_y is None else d_y
    back = zero.clone() if d_state is None else d_state.clone()
    back_size = back.abs()
    whole, whole_size = torch.zeros_like(x), torch.zeros_like(x)
    for d, rows in enumerate(order):
        for t in reversed(rows):
            whole[t] = d_y[t] * open_[t] + back[d]
            whole_size[t] = (d_y[t] * open_[t]).abs() + back_size[d]
            back[d], back_size[d] = a[t] * whole[t], a[t] * whole_size[t]
    value.update(d_x=whole * rest, d_forget=whole * (before - x) * a * rest, d_initial=back)
    size.update(d_x=whole_size * rest, d_forget=whole_size * (before_size + x.abs()) * a * rest, d_initial=back_size)
    if o is not None:
        value["d_gate"] = d_y * after * (p + o * p * (1 - p))
        size["d_gate"] = d_y.abs() * after_size * (p + o.abs() * p * (1 - p))
    return value, size


# ---- projections -------------------------------------------------------------------------------------


def activate(z, how):
    """act(z), act'(z)."""
    if how == "none":
        return z, torch.ones_like(z)
    if how == "relu":
        return z.clamp(min=0), (z > 0).double()
    if how == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if how == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = 2 * math.sqrt(2 / math.pi)
    p = torch.sigmoid(a * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * a * (1 + 3 * 0.044715 * z * z)


CURVE = {"none": 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.8}  # the largest |act''|


def linear(x, weight, bias=None, activation="none", residual=None, d_out=None):
    x, w, bias, residual, d_out = map(wide, (x, weight, bias, residual, d_out))
    z, z_size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, z_size = z + bias, z_size + bias.abs()
    out, slope = activate(z, activation)
    value, size = {"z": z, "out": out}, {"z": z_size, "out": out.abs()}
    if residual is not None:
        value["out"], size["out"] = out + residual, out.abs() + residual.abs()
    if d_out is not None:
        d = d_out * slope
        value.update(dz=d, d_x=d @ w, d_weight=d.t() @ x, d_bias=d.sum(0))
        size.update(dz=d.abs(), d_x=d.abs() @ w.abs(), d_weight=d.abs().t() @ x.abs(), d_bias=d.abs().sum(0))
    return value, size
