"""Linear attention with a decay for each head, token by token in 64 bits, with its gradients by their formulas."""

from __future__ import annotations

import torch


def forward(q, k, v, g, scale=1.0, h0=None, lengths=None):
    """y and the state after each token, (batch, seqlen + 1, heads, key_dim, value_dim), the first one h0."""
    q, k, v = (t.double() for t in (q, k, v))
    b, n, heads, dv = v.shape
    per = heads // q.shape[2]
    q, k = q.repeat_interleave(per, 2), k.repeat_interleave(per, 2)
    g = g.double().expand(b, n, heads)
    h = v.new_zeros((b, heads, q.shape[3], dv)) if h0 is None else h0.double()
    ends = torch.full((b,), n) if lengths is None else lengths.long().clamp(0, n)
    ends = ends.to(v.device)
    y, states = torch.zeros_like(v), [h]
    for t in range(n):
        on = (ends > t)[:, None, None]
        new = torch.exp(g[:, t])[..., None, None] * h + k[:, t][..., None] * v[:, t][..., None, :]
        h = torch.where(on[..., None], new, h)
        y[:, t] = torch.where(on, scale * (q[:, t][..., None] * h).sum(2), torch.zeros_like(y[:, t]))
        states.append(h)
    return y, torch.stack(states, 1)


def backward(q, k, v, g, dy, scale=1.0, h0=None, lengths=None, dstate=None):
    """dq, dk, dv, dg (batch, seqlen, heads) and dh0."""
    _, states = forward(q, k, v, g, scale, h0, lengths)
    q, k, v, dy = (t.double() for t in (q, k, v, dy))
    b, n, heads, dv_ = v.shape
    groups = q.shape[2]
    per = heads // groups
    qh, kh = q.repeat_interleave(per, 2), k.repeat_interleave(per, 2)
    a = torch.exp(g.double().expand(b, n, heads))
    ends = (torch.full((b,), n) if lengths is None else lengths.long().clamp(0, n)).to(v.device)
    dS = torch.zeros_like(states[:, 0]) if dstate is None else dstate.double()
    dq, dk = torch.zeros_like(qh), torch.zeros_like(kh)
    dv, dg = torch.zeros_like(v), torch.zeros_like(a)
    zero = torch.zeros((), dtype=torch.float64, device=v.device)
    for t in range(n - 1, -1, -1):
        on = (ends > t)[:, None, None]
        here = dS + scale * qh[:, t][..., None] * dy[:, t][..., None, :]
        dq[:, t] = torch.where(on, scale * (states[:, t + 1] * dy[:, t][..., None, :]).sum(3), zero)
        dk[:, t] = torch.where(on, (here * v[:, t][..., None, :]).sum(3), zero)
        dv[:, t] = torch.where(on, (here * kh[:, t][..., None]).sum(2), zero)
        dg[:, t] = torch.where(on[..., 0], a[:, t] * (here * states[:, t]).sum((2, 3)), zero)
        dS = torch.where(on[..., None], a[:, t][..., None, None] * here, dS)
    shared = lambda t: t.view(b, n, groups, per, -1).sum(3)
    return shared(dq), shared(dk), dv, dg, dS
