"""The selective state space block in 64 bits, written from its formulas: results and gradients of the convolution, the scan and
the norms, on the CPU.  With ``absolute`` every term of a sum counts with its absolute value, which is what the errors of the sums are
measured against."""
import torch

EPS32 = 2.0 ** -24      # half a step of fp32 at 1


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of the type's smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def double(t):
    return None if t is None else t.detach().cpu().double()


def alive(lengths, N, L):
    n = torch.full((N,), L) if lengths is None else lengths.cpu()
    return (torch.arange(L) < n[:, None])[:, None, :, None]


def silu_slope(x):
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def conv(x, w, b, state=None, silu=False, lengths=None, gy=None, absolute=False):
    """(y, the last K-1 rows) or, with gy, also (gx, gw, gb)"""
    N, H, L, D = x.shape
    K = w.shape[-1]
    live = alive(lengths, N, L)
    x = torch.where(live, x, 0.0)
    first = torch.zeros(N, H, K - 1, D, dtype=torch.float64) if state is None else state
    ext = torch.cat([first, x], 2)
    taps = [ext[:, :, j:j + L] for j in range(K)]
    p = sum(w[:, None, :, j] * taps[j] for j in range(K)) + (0 if b is None else b[:, None])
    if absolute:
        y = sum((w[:, None, :, j] * taps[j]).abs() for j in range(K)) + (0 if b is None else b[:, None].abs())
    else:
        y = p * torch.sigmoid(p) if silu else p
    n = torch.full((N,), L) if lengths is None else lengths.cpu().clamp(0, L)
    last = torch.stack([ext[i, :, n[i]:n[i] + K - 1] for i in range(N)])
    y = torch.where(live, y, 0.0)
    if gy is None:
        return y, last
    d = torch.where(live, gy, 0.0) * (silu_slope(p) if silu else 1.0)
    if absolute:        # the slope of the activation moves by at most half of what p is off, and p by parts of its terms
        d = torch.where(live, gy, 0.0).abs() * (1.1 + y if silu else 1.0)
    ab = torch.abs if absolute else (lambda t: t)
    after = torch.cat([d, torch.zeros(N, H, K - 1, D, dtype=torch.float64)], 2)
    gx = sum(ab(w[:, None, :, j]) * after[:, :, K - 1 - j:K - 1 - j + L] for j in range(K))
    gw = torch.stack([ab(d * taps[j]).sum((0, 2)) for j in range(K)], -1)
    return y, last, torch.where(live, gx, 0.0), gw, d.sum((0, 2))


def scan(q, k, v, delta, A, W=None, D=None, z=None, bias=None, softplus=False, lengths=None, go=None, absolute=False):
    """(out, the last state) or, with go, also the gradients of q, k, v, delta, A, D, z, bias"""
    N, H, L, E = q.shape
    M = v.shape[-1]
    live = alive(lengths, N, L)
    q, k, v, delta = (torch.where(live, t, 0.0) for t in (q, k, v, delta))
    z = None if z is None else torch.where(live, z, 0.0)
    ab = torch.abs if absolute else (lambda t: t)
    q, k, v = ab(q), ab(k), ab(v)
    D = torch.zeros(H, M, dtype=torch.float64) if D is None else ab(D)
    pre = delta if bias is None else delta + bias[:, None]
    dt = torch.where(live, torch.nn.functional.softplus(pre, threshold=700) if softplus else pre, 0.0)
    x = ab(dt) * v
    gate = 1.0 if z is None else z * torch.sigmoid(z)
    state = torch.zeros(N, H, E, M, dtype=torch.float64) if W is None else ab(W)
    decay, states = torch.exp(dt[:, :, :, None] * A[:, None]), []
    for t in range(L):
        state = decay[:, :, t] * state + k[:, :, t, :, None] * x[:, :, t, None]
        states.append(state)
    h = torch.stack(states, 2)
    o = (q[..., None] * h).sum(-2) + D[:, None] * v
    out = torch.where(live, o * ab(torch.as_tensor(gate)), 0.0)
    if go is None:
        return out, state
    go = torch.where(live, go, 0.0)
    dy = ab(go * gate)
    before = torch.cat([(torch.zeros(N, H, 1, E, M, dtype=torch.float64) if W is None else ab(W)[:, :, None]), h[:, :, :-1]], 2)
    c, gs = torch.zeros(N, H, E, M, dtype=torch.float64), [None] * L
    for t in reversed(range(L)):
        gs[t] = dy[:, :, t, None] * q[:, :, t, :, None] + c
        c = decay[:, :, t] * gs[t]
    g = torch.stack(gs, 2)
    read, w = (g * k[..., None]).sum(-2), g * decay * before
    gdt = v * read + (w * ab(A[:, None])).sum(-2)
    gdelta = torch.where(live, gdt * torch.sigmoid(pre) if softplus else gdt, 0.0)
    if z is None:
        gz = None
    elif absolute:      # the slope s (1 + z (1 - s)) with its terms positive: near its zero at z = -1.28 they cancel
        s = torch.sigmoid(z)
        gz = go.abs() * s * (1 + z.abs() * (1 - s)) * o
    else:
        gz = go * silu_slope(z) * o
    return (out, state, (h * dy[..., None, :]).sum(-1), (g * x[..., None, :]).sum(-1), ab(dt) * read + D[:, None] * dy, gdelta,
            (w * ab(dt)[:, :, :, None]).sum((0, 2)), (dy * v).sum((0, 2)), gz, gdelta.sum((0, 2)))


def activation(g, act):
    return g if act is None else torch.sigmoid(g) if act == "sigmoid" else g * torch.sigmoid(g)


def residual_norm(y, x, aw=None, ab=None, gate=None, scale=None, bw=None, bb=None, eps=1e-5, rms=False, act=None):
    """(r, n); its gradients are autograd's"""
    def norm(t, w, b):
        if w is None:
            return t
        t = t if rms else t - t.mean(-1, keepdim=True)
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w
        return t if b is None else t + b
    u = norm(y, aw, ab)
    u = u if gate is None else u * activation(gate, act)
    r = x + (u if scale is None else scale * u)
    return r, None if bw is None else norm(r, bw, bb)
