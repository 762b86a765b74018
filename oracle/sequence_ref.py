"""Oracle of the sequence operators: their definitions in float64, on any device.

Layer norm, rotary positions over several axes, and linear attention with a
decay for each head as its recurrence, token by token, with the gradients
written out as recurrences too (not by autograd, not in chunks).
"""
from __future__ import annotations

import torch


def layer_norm(x, weight=None, bias=None, eps=1e-5, dy=None):
    """y, and (dx, dweight, dbias) if dy is given."""
    x = x.double()
    n = x.size(-1)
    c = x - x.sum(-1, keepdim=True) / n
    rstd = (c.square().sum(-1, keepdim=True) / n + eps).rsqrt()
    xhat = c * rstd
    w = 1.0 if weight is None else weight.double()
    y = xhat * w + (0.0 if bias is None else bias.double())
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return y, (dx, (dy * xhat).sum(lead), dy.sum(lead))


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    """x [.., H, D] turned by positions [.., A]."""
    x = x.double().clone()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[..., axis] * inv_freq)[..., None, :]
    if inverse:
        angle = -angle
    P = len(axis)
    if interleaved:
        u, v = x[..., 0:2 * P:2].clone(), x[..., 1:2 * P:2].clone()
    else:
        u, v = x[..., :P].clone(), x[..., P:2 * P].clone()
    a, b = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
    if interleaved:
        x[..., 0:2 * P:2], x[..., 1:2 * P:2] = a, b
    else:
        x[..., :P], x[..., P:2 * P] = a, b
    return x


def decay_attention(q, k, v, log_decay, scale, state=None, lengths=None, do=None, dstate=None):
    """(out, state), and (dq, dk, dv, dstate0) if do is given."""
    B, T, H, Dk = q.shape
    Hk, Dv = k.size(2), v.size(3)
    group = H // Hk
    dev = q.device
    q = q.double()
    k, v = (t.double().repeat_interleave(group, 2) for t in (k, v))
    g = log_decay.double().exp().view(1, H, 1, 1)
    lens = torch.full((B,), T, device=dev) if lengths is None else lengths.to(dev).long().clamp(0, T)
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=dev) if state is None else state.double().clone()
    S0 = S
    out = torch.zeros(B, T, H, Dv, dtype=torch.float64, device=dev)
    dq = torch.zeros(B, T, H, Dk, dtype=torch.float64, device=dev)
    do = None if do is None else do.double()
    for t in range(T):
        on = (t < lens)
        new = S * g + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(on.view(B, 1, 1, 1), new, S)
        o = scale * (q[:, t, :, :, None] * S).sum(-2)
        out[:, t] = torch.where(on.view(B, 1, 1), o, torch.zeros_like(o))
        if do is not None:
            d = scale * (S * do[:, t, :, None, :]).sum(-1)
            dq[:, t] = torch.where(on.view(B, 1, 1), d, torch.zeros_like(d))
    if do is None:
        return out, S
    G = torch.zeros_like(S0) if dstate is None else dstate.double().clone()
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T - 1, -1, -1):
        on = (t < lens)
        now = G + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        a = (now * v[:, t, :, None, :]).sum(-1)
        b = (now * k[:, t, :, :, None]).sum(-2)
        dk[:, t] = torch.where(on.view(B, 1, 1), a, torch.zeros_like(a))
        dv[:, t] = torch.where(on.view(B, 1, 1), b, torch.zeros_like(b))
        G = torch.where(on.view(B, 1, 1, 1), now * g, G)
    dk = dk.view(B, T, Hk, group, Dk).sum(3)
    dv = dv.view(B, T, Hk, group, Dv).sum(3)
    return (out, S), (dq, dk, dv, G)
