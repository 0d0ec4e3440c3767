"""The decayed sum rule, rotary positions and the norm of groups of channels in 64 bits, written from their formulas, on the CPU.  With ``absolute`` every term of a sum
counts with its absolute value, which is what the errors of the sums are measured against."""
import math

import torch

from scan_formulas import EPS32, alive, double, half_step, smallest      # noqa: F401 (what the tests go by)


def shared(t, H):
    """[N,G,L,D] as [N,H,L,D]: head h takes head h // (H // G)"""
    return t.repeat_interleave(H // t.shape[1], 1)


def decayed_sum(q, k, v, g, W=None, scale=1.0, lengths=None, go=None, absolute=False, reach=64):
    """(out, the last state) or, with go, also the gradients of q, k, v and g, step by step.

    The size of a decay's gradient: of all that the steps from this one on, within `reach` of them, read and wrote, and of what is read beyond them of what was
    written before."""
    N, L, H = q.shape[0], q.shape[2], g.shape[-1] if g.dim() == 1 else g.shape[1]
    per_head = g.dim() == 1
    live = alive(lengths, N, L)
    G = [t.shape[1] for t in (q, k, v)]
    q, k, v = (shared(torch.where(live, t, 0.0), H) for t in (q, k, v))
    g = g[None, :, None].expand(N, H, L) if per_head else g
    a = torch.where(live[..., 0], torch.exp(g), 1.0)
    ab = torch.abs if absolute else (lambda t: t)
    q, k, v = ab(q) * scale, ab(k), ab(v)
    S = torch.zeros(N, H, q.shape[-1], v.shape[-1], dtype=torch.float64) if W is None else ab(W)
    before, after = [], []
    for t in range(L):
        before.append(S)
        S = a[:, :, t, None, None] * S + k[:, :, t, :, None] * v[:, :, t, None, :]
        after.append(S)
    h = torch.stack(after, 2)
    out = torch.where(live, (q[..., None] * h).sum(-2), 0.0)
    if go is None:
        return out, S
    go = ab(torch.where(live, go, 0.0))
    c, adj = torch.zeros_like(S), [None] * L
    through = [None] * L
    for t in reversed(range(L)):
        through[t] = (c * after[t]).sum((-1, -2))
        adj[t] = c + q[:, :, t, :, None] * go[:, :, t, None, :]
        c = a[:, :, t, None, None] * adj[t]
    d = torch.stack(adj, 2)
    gq, gk, gv = (h * go[..., None, :]).sum(-1) * scale, (d * v[..., None, :]).sum(-1), (d * k[..., None]).sum(-2)
    if absolute:
        rows = (q * gq / scale).sum(-1) + (k * gk).sum(-1)
        far = torch.stack(through, 2)
        pad = lambda t: torch.cat([t, torch.zeros(N, H, reach - 1, dtype=t.dtype)], 2).unfold(2, reach, 1)
        gg = pad(rows).sum(-1) + pad(far).amax(-1)
    else:
        gg = (d * a[..., None, None] * torch.stack(before, 2)).sum((-1, -2))
    gg = torch.where(live[..., 0], gg, 0.0)
    back = lambda t, n: torch.where(live, t, 0.0).view(N, n, H // n, L, t.shape[-1]).sum(2)
    return out, S, back(gq, G[0]), back(gk, G[1]), back(gv, G[2]), gg.sum((0, 2)) if per_head else gg


def rotary(x, frequencies, positions=None, interleaved=False, scale=1.0, lengths=None, absolute=False):
    """The turned rows; ``absolute``: (|a| + |b|) scale for both of a pair"""
    N, H, L, D = x.shape
    n = len(frequencies)
    x = torch.where(alive(lengths, N, L), x, 0.0)
    at = torch.arange(L).expand(N, L)
    if positions is not None:
        at = positions if positions.dim() == 2 else at + positions[:, None]
    angle = at[:, None, :, None].double() * frequencies.double()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    if absolute:
        p, r = 2 * [(a.abs() + b.abs()) * scale]
    else:
        p, r = scale * (a * torch.cos(angle) - b * torch.sin(angle)), scale * (a * torch.sin(angle) + b * torch.cos(angle))
    y = torch.stack([p, r], -1).flatten(-2) if interleaved else torch.cat([p, r], -1)
    return torch.cat([y, x[..., 2 * n:].abs() if absolute else x[..., 2 * n:]], -1)


def act(x, name):
    return x if name is None else torch.sigmoid(x) if name == "sigmoid" else x * torch.sigmoid(x)


def group_norm(x, groups, w=None, b=None, gate=None, eps=1e-5, rms=False, activation=None):
    """Its gradients are autograd's"""
    t = x.unflatten(-1, (groups, -1))
    t = t if rms else t - t.mean(-1, keepdim=True)
    u = (t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)).flatten(-2)
    u = u if w is None else u * w
    u = u if b is None else u + b
    return act(u, activation) if gate is None else u * act(gate, activation)


def frequencies(width, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / width) for i in range(width // 2)], dtype=torch.float64)


def turns_per(trained, f):
    return trained * f / (2 * math.pi)
