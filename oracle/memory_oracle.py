"""Plain restatement in float64 of the memory policy's operators: decayed linear attention token by token, group norm
with an activation, their gradients from the formulas, and the size of what is summed (for error bounds)."""
from __future__ import annotations

import torch


def attn_forward(q, k, v, log_decay, reset=None, state=None, scale=1.0):
    """q, k, v (N, T, H, D) float64; returns o, the last state, and the state after every token (list)."""
    n, t, h, d = q.shape
    lam = torch.exp(log_decay)[None, :, None, None]
    s = torch.zeros(n, h, d, d, dtype=q.dtype) if state is None else state.clone()
    o, states = torch.empty_like(q), []
    for i in range(t):
        s = s * lam
        if reset is not None:
            s = torch.where(reset[:, i, None, None, None].bool(), torch.zeros_like(s), s)
        s = s + k[:, i, :, :, None] * v[:, i, :, None, :]
        o[:, i] = scale * torch.einsum("nhi,nhij->nhj", q[:, i], s)
        states.append(s)
    return o, s, states


def attn_backward(q, k, v, log_decay, do, reset=None, state=None, dlast=None, scale=1.0):
    """dq, dk, dv and the gradient of the first state."""
    n, t, h, d = q.shape
    lam = torch.exp(log_decay)[None, :, None, None]
    _, _, states = attn_forward(q, k, v, log_decay, reset, state, scale)
    u = torch.zeros(n, h, d, d, dtype=q.dtype) if dlast is None else dlast.clone()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    for i in reversed(range(t)):
        u = u + scale * q[:, i, :, :, None] * do[:, i, :, None, :]
        dq[:, i] = scale * torch.einsum("nhj,nhij->nhi", do[:, i], states[i])
        dk[:, i] = torch.einsum("nhj,nhij->nhi", v[:, i], u)
        dv[:, i] = torch.einsum("nhi,nhij->nhj", k[:, i], u)
        u = u * lam
        if reset is not None:
            u = torch.where(reset[:, i, None, None, None].bool(), torch.zeros_like(u), u)
    return dq, dk, dv, u


def act(z, name):
    return z * torch.sigmoid(z) if name == "silu" else z.clamp(min=0) if name == "relu" else z


def norm_parts(x, groups, eps):
    """x (N, C, P) float64: mean, rstd (N, G, 1, 1) and x as (N, G, C/G, P)."""
    n, c, p = x.shape
    xg = x.reshape(n, groups, c // groups, p)
    mean = xg.mean((2, 3), keepdim=True)
    return xg, mean, ((xg - mean).square().mean((2, 3), keepdim=True) + eps).rsqrt()


def norm_forward(x, groups, w, b, eps, name):
    xg, mean, rstd = norm_parts(x, groups, eps)
    return act(((xg - mean) * rstd).reshape(x.shape) * w[None, :, None] + b[None, :, None], name)


def codes(x, groups):
    """x (N, C, P) float32: the 8-bit codes' values, by the 32-bit rule."""
    n, c, p = x.shape
    xg = x.reshape(n, groups, -1)
    lo, hi = xg.amin(-1, keepdim=True), xg.amax(-1, keepdim=True)
    q = torch.round((xg - lo) * torch.where(hi > lo, 255.0 / (hi - lo), torch.zeros_like(lo)))
    return (lo + q * ((hi - lo) / 255.0)).reshape(x.shape)


def norm_backward(x, groups, w, b, eps, name, dy, kept=None):
    """dx, dw, db (N, C, P), (C,), (C,); kept: what stands for x in the backward pass."""
    n, c, p = x.shape
    xg, mean, rstd = norm_parts(x, groups, eps)
    kg = xg if kept is None else kept.reshape(xg.shape)
    xh = (kg - mean) * rstd
    z = xh.reshape(x.shape) * w[None, :, None] + b[None, :, None]
    if name == "silu":
        s = torch.sigmoid(z)
        dz = dy * s * (1 + z * (1 - s))
    else:
        dz = torch.where(z <= 0, torch.zeros_like(dy), dy) if name == "relu" else dy
    dw, db = (dz * xh.reshape(x.shape)).sum((0, 2)), dz.sum((0, 2))
    dh = (dz * w[None, :, None]).reshape(xg.shape)
    dx = rstd * (dh - dh.mean((2, 3), keepdim=True) - xh * (dh * xh).mean((2, 3), keepdim=True))
    return dx.reshape(x.shape), dw, db
