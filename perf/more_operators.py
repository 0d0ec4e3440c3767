"""The operators of a block whose fast weights decay, as they are measured: the sum rule with a decay for each head, rotary positions
of its queries and keys, and the norm of every head's channels with its gate.

    own                   False: run() computes the plain form, elementary torch operations; True: the framework's operators
    listed()              the cases by name
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   what a program holds before the call: inputs, parameters, the state it carries
    run(state)            one pass through an operator, and its results
    work(case)            bytes and operations that one pass cannot do without
    exact(case, seed)     what run() returns, from the definition in 64 bits

A case's mode: "train" (forward and backward of one call), "forward" (a prompt: nothing recorded, the state kept), "step" (one
token per sequence, the state advanced in place).
"""
import importlib
import math

import torch
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _sum(mode, N, H, L, E, M, dtype, G=None, token_decay=False, ragged=False, time_major=False):
    """H heads of values and decays, G heads of queries and keys that H / G of them share."""
    return dict(op="sum", mode=mode, N=N, H=H, G=G or H, L=L, E=E, M=M, dtype=dtype, token_decay=token_decay, ragged=ragged, time_major=time_major)


def _rotary(mode, N, H, G, L, D, width, dtype, interleaved=False, scaling="none", ragged=False, time_major=False):
    """H heads of queries and G of keys, D channels each of which the first `width` turn."""
    return dict(op="rotary", mode=mode, N=N, H=H, G=G, L=L, D=D, width=width, dtype=dtype, interleaved=interleaved, scaling=scaling,
                ragged=ragged, time_major=time_major)


def _norm(mode, rows, groups, size, dtype, rms=False, gated=True, affine=True):
    return dict(op="norm", mode=mode, rows=rows, groups=groups, size=size, dtype=dtype, rms=rms, gated=gated, affine=affine)


def listed():
    return [
        # decoding: one token for each of 32 sequences of a model with d_model 256, 8 heads
        dict(_sum("step", 32, 8, 1, 32, 32, "fp32"), name="sum_step"),
        # decoding for many users of a wider model: bound by the state's bytes
        dict(_sum("step", 256, 16, 1, 128, 128, "bf16", token_decay=True), name="sum_step_many"),
        # one long prompt: few heads, all of the parallelism has to come from the sequence
        dict(_sum("forward", 1, 8, 16384, 64, 64, "bf16", token_decay=True), name="sum_prompt"),
        # prompts of different lengths in one padded batch, heads that share queries and keys, widths that are no multiple of anything
        dict(_sum("forward", 7, 6, 1531, 41, 73, "fp16", G=2, token_decay=True, ragged=True), name="sum_prompt_ragged"),
        # one layer of the language model's training step: 32 x 1024 tokens, tensors as a layer hands them over
        dict(_sum("train", 32, 8, 1024, 32, 32, "fp32", time_major=True), name="sum_train"),
        # a wider model's training step on long sequences
        dict(_sum("train", 8, 16, 4096, 64, 64, "bf16", token_decay=True, time_major=True), name="sum_train_wide"),
        # all heads share one wide pair of queries and keys, as in a state space model
        dict(_sum("train", 4, 32, 4096, 128, 64, "bf16", G=1, token_decay=True, time_major=True), name="sum_train_shared"),
        # decoding: the queries and keys of one token for each of 32 sequences, at positions of their own
        dict(_rotary("step", 32, 8, 8, 1, 32, 32, "fp32"), name="rotary_step"),
        # one layer of the language model's training step
        dict(_rotary("train", 32, 8, 8, 1024, 32, 32, "fp32", time_major=True), name="rotary_train"),
        # a long prompt far behind the trained length: half of every head turns, fewer heads of keys than of queries
        dict(_rotary("forward", 1, 32, 8, 32768, 128, 64, "bf16", interleaved=True, scaling="parts", time_major=True), name="rotary_prompt"),
        # one layer of the language model's training step: the norm of 8 heads, gated
        dict(_norm("train", 32768, 8, 32, "fp32"), name="norm_train"),
        # a wide model in bf16
        dict(_norm("train", 16384, 32, 128, "bf16", rms=True), name="norm_train_wide"),
    ]


def _between(rng, lo, hi):
    """A whole number from [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("sum", "sum", "sum", "rotary", "norm"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op == "norm":
        groups, size = rng.choice((1, 2, 4, 8, 16, 32, _between(rng, 1, 48))), rng.choice((16, 32, 64, 128, _between(rng, 3, 256)))
        groups = min(groups, 8192 // size)
        rows = _between(rng, 1, max(1, min(65536, (1 << 26) // (groups * size))))
        return _norm(rng.choice(("train", "train", "forward")), rows, groups, size, dtype, rng.random() < 0.5, rng.random() < 0.7,
                     rng.random() < 0.7)
    mode = rng.choice(("train", "train", "forward", "step"))
    ragged, time_major = mode != "step" and rng.random() < 0.3, rng.random() < 0.5
    if op == "rotary":
        D = rng.choice((32, 64, 128, 256, 2 * _between(rng, 4, 128)))
        width = rng.choice((D, D, 2 * max(1, D // 4), 2 * rng.randint(1, D // 2)))
        G = rng.choice((1, 2, 4, 8))
        H = G * rng.choice((1, 2, 4))
        L = 1 if mode == "step" else _between(rng, 2, 16384)
        N = _between(rng, 1, max(1, min(256, (1 << 26) // (L * (H + G) * D))))
        return _rotary(mode, N, H, G, L, D, width, dtype, rng.random() < 0.5, rng.choice(("none", "linear", "base", "parts")), ragged, time_major)
    H = rng.choice((1, 2, 4, 8, 16, 32, rng.randint(1, 24)))
    G = rng.choice((H, H, H, 1, math.gcd(H, 4)))
    E = rng.choice((16, 32, 64, 128, _between(rng, 1, 128)))
    M = rng.choice((16, 32, 64, 128, _between(rng, 1, 256)))
    L = 1 if mode == "step" else _between(rng, 2, 16384)
    cells = H * max(E, 16) * max(M, 16)
    L = min(L, max(1, (1 << 31) // cells))
    N = _between(rng, 1, max(1, min(256, (1 << 31) // (cells * L), (1 << 26) // cells, (1 << 26) // (L * H * (E + M)))))
    return _sum(mode, N, H, L, E, M, dtype, G, rng.random() < 0.6, ragged, time_major)


# ------------------------------------------------------------------ inputs

def _rows(g, case, heads, width):
    """N(0,1) values [N,heads,L,width], or the permuted view of [L,N,heads,width] storage that a layer has."""
    N, L = case["N"], case["L"]
    shape = (L, N, heads, width) if case["time_major"] else (N, heads, L, width)
    x = torch.randn(shape, generator=g, device="cuda").to(TYPES[case["dtype"]])
    return x.permute(1, 2, 0, 3) if case["time_major"] else x


def _lengths(g, case):
    """One sequence is whole, one is empty where there are three, the others end anywhere."""
    if not case["ragged"]:
        return None
    n = torch.randint(1, case["L"] + 1, (case["N"],), generator=g, device="cuda")
    n[0] = case["L"]
    if case["N"] > 2:
        n[2] = 0
    return n


def _prepare_sum(case, g):
    N, H, G, L, E, M = (case[k] for k in ("N", "H", "G", "L", "E", "M"))
    s = dict(q=_rows(g, case, G, E), k=_rows(g, case, G, E), v=_rows(g, case, H, M), lengths=_lengths(g, case), scale=E ** -0.5)
    if case["token_decay"]:
        # every head has a rate of its own, from memories of a few tokens to some of a thousand, which the token moves
        rate = torch.exp(torch.empty(H, 1, device="cuda").uniform_(math.log(1e-3), 0.0, generator=g))
        x = torch.randn(N, H, L, generator=g, device="cuda")
        s["decay"] = -rate * (torch.log1p(torch.exp(-x.abs())) + x.clamp(min=0))
    else:
        # one rate a head: a memory of 32 tokens for the first, twice as long for each one behind it, not beyond some 4000
        s["decay"] = torch.log1p(-torch.exp2(-5.0 - torch.arange(H, device="cuda").clamp(max=7)))
        s["decay"] = s["decay"] * (1 + 0.1 * torch.rand(H, generator=g, device="cuda"))
    s["W"] = None if case["mode"] == "train" else torch.randn(N, H, E, M, generator=g, device="cuda")
    s["diff"] = ["q", "k", "v", "decay"]
    s["grads"] = [_rows(g, case, H, M)] if case["mode"] == "train" else None
    return s


def _frequencies(case):
    """Radians a position for every pair, and the factor of the rotated rows, for contexts 8 times as long as those of training."""
    width, base, factor, trained, scale = case["width"], 10000.0, 8.0, 4096, 1.0
    pair = torch.arange(width // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "base":
        base *= factor ** (width / max(width - 2, 1))
    f = base ** (-2.0 * pair / width)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":
        # pairs that turn more than 32 times over the trained length stay, those that turn less than once are slowed down
        kept = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, scale = f * (kept + (1 - kept) / factor), 1 + 0.1 * math.log(factor)
    return f, scale


def _prepare_rotary(case, g):
    N, L = case["N"], case["L"]
    s = dict(q=_rows(g, case, case["H"], case["D"]), k=_rows(g, case, case["G"], case["D"]), lengths=_lengths(g, case))
    s["frequencies"], s["scale"] = _frequencies(case)
    # training starts at the sequence's start, a prompt and a token anywhere behind what came before
    far = 4096 if case["scaling"] == "none" else 1 << 20
    s["positions"] = None if case["mode"] == "train" else torch.randint(0, far, (N,), generator=g, device="cuda")
    s["diff"] = ["q", "k"]
    s["grads"] = [_rows(g, case, case["H"], case["D"]), _rows(g, case, case["G"], case["D"])] if case["mode"] == "train" else None
    return s


def _prepare_norm(case, g):
    R, C, T = case["rows"], case["groups"] * case["size"], TYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    s = dict(x=(0.5 * normal(R, C) + 0.1).to(T), gate=normal(R, C).to(T) if case["gated"] else None)
    s["weight"] = 1 + 0.1 * normal(C) if case["affine"] else None
    s["bias"] = 0.1 * normal(C) if case["affine"] and not case["rms"] else None
    s["diff"] = [k for k in ("x", "weight", "bias", "gate") if s[k] is not None]
    s["grads"] = [normal(R, C).to(T)]
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"sum": _prepare_sum, "rotary": _prepare_rotary, "norm": _prepare_norm}[case["op"]](case, g)
    s["case"] = case
    if case["mode"] == "train":
        for k in s["diff"]:
            s[k] = s[k].detach().requires_grad_()
    return s


# ------------------------------------------------------------------ the plain forms

def _valid(s):
    """[N,1,L,1]: is this row one of its sequence's (None: all are)?"""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["L"], device="cuda") < s["lengths"][:, None])[:, None, :, None]


def _masked(t, valid):
    return t if valid is None else torch.where(valid, t, torch.zeros((), device=t.device, dtype=t.dtype))


BLOCK = 128


def _plain_sum(s):
    """Blocks of steps: products within a block, and with the state that the blocks before it have left."""
    case, T = s["case"], s["v"].dtype
    N, H, G, L, E, M = (case[k] for k in ("N", "H", "G", "L", "E", "M"))
    valid, R = _valid(s), H // G
    each = lambda t: _masked(t.float(), valid).repeat_interleave(R, 1)                # a copy for each head that shares it
    q, k, v = each(s["q"]) * s["scale"], each(s["k"]), _masked(s["v"].float(), valid)
    decay = s["decay"].double()
    decay = decay[None, :, None].expand(N, H, L) if decay.dim() == 1 else decay
    decay = _masked(decay[..., None], valid)[..., 0]
    blocks = []
    W = torch.zeros(N, H, E, M, device="cuda") if s["W"] is None else s["W"]
    outs = []
    for i in range(0, L, BLOCK):
        qi, ki, vi = (t[:, :, i:i + BLOCK] for t in (q, k, v))
        b = decay[:, :, i:i + BLOCK].cumsum(-1)
        apart = torch.exp((b[..., :, None] - b[..., None, :]).tril()).float().tril()
        into, rest, whole = torch.exp(b).float()[..., None], torch.exp(b[..., -1:] - b).float()[..., None], torch.exp(b[..., -1]).float()[..., None, None]
        p = torch.matmul(qi, ki.transpose(-1, -2)) * apart
        outs.append(torch.matmul(p, vi) + into * torch.matmul(qi, W))
        after = whole * W + torch.matmul(ki.transpose(-1, -2), rest * vi)
        blocks.append((i, apart, into, rest, whole, W, after))
        W = after
    out = torch.cat(outs, 2).to(T)
    if s["W"] is not None:
        s["W"].copy_(W)
        return [out, s["W"]]
    do = _masked(s["grads"][0].float(), valid)
    adjoint = torch.zeros_like(W)
    gq, gk, gv, gdecay = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty(N, H, L, device="cuda")
    for i, apart, into, rest, whole, before, after in reversed(blocks):
        qi, ki, vi, di = (t[:, :, i:i + BLOCK] for t in (q, k, v, do))
        p = torch.matmul(qi, ki.transpose(-1, -2)) * apart
        r = torch.matmul(di, vi.transpose(-1, -2)) * apart
        dq = torch.matmul(r, ki) + into * torch.matmul(di, before.transpose(-1, -2))
        dk = torch.matmul(r.transpose(-1, -2), qi) + rest * torch.matmul(vi, adjoint.transpose(-1, -2))
        gv[:, :, i:i + BLOCK] = torch.matmul(p.transpose(-1, -2), di) + rest * torch.matmul(ki, adjoint)
        gq[:, :, i:i + BLOCK], gk[:, :, i:i + BLOCK] = dq, dk
        # a step's decay scales all that came before it: what is read from there on but was not written from there on
        here = ((qi * dq).sum(-1) - (ki * dk).sum(-1)).flip(-1).cumsum(-1).flip(-1)
        gdecay[:, :, i:i + BLOCK] = here + (adjoint * after).sum((-1, -2))[..., None]
        adjoint = whole * adjoint + torch.matmul((into * qi).transpose(-1, -2), di)
    shared = lambda t: _masked(t.view(N, G, R, L, E).sum(2), valid).to(T)
    gdecay = _masked(gdecay[..., None], valid)[..., 0]
    return [out, shared(gq * s["scale"]), shared(gk), gv.to(T), gdecay.sum((0, 2)) if s["decay"].dim() == 1 else gdecay]


def _turned(x, cos, sin, case, valid):
    """The first `width` channels of every row turned, the others as they are."""
    T, w = x.dtype, case["width"]
    x = _masked(x.float(), valid)
    if case["interleaved"]:
        a, b = x[..., 0:w:2], x[..., 1:w:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :w // 2], x[..., w // 2:w]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., w:]], -1).to(T)


def _plain_rotary(s):
    case, valid = s["case"], _valid(s)
    at = torch.arange(case["L"], device="cuda")[None]
    if s["positions"] is not None:
        at = at + s["positions"][:, None]
    angle = at[:, None, :, None].double() * s["frequencies"]                          # far angles need 64 bits
    cos, sin = (s["scale"] * f(angle).float() for f in (torch.cos, torch.sin))
    res = [_turned(s[n], cos, sin, case, valid) for n in ("q", "k")]
    if case["mode"] == "train":
        res += [_turned(g, cos, -sin, case, valid) for g in s["grads"]]
    return res


EPS = 1e-5


def _plain_norm(s):
    case, T = s["case"], s["x"].dtype
    R, G, D = case["rows"], case["groups"], case["size"]
    x = s["x"].float().view(R, G, D)
    xc = x if case["rms"] else x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    w = None if s["weight"] is None else s["weight"].view(G, D)
    u = xh if w is None else xh * w
    if s["bias"] is not None:
        u = u + s["bias"].view(G, D)
    gate = None if s["gate"] is None else s["gate"].float().view(R, G, D)
    at = u if gate is None else gate
    sig = torch.sigmoid(at)
    y = (at * sig if gate is None else u * at * sig).view(R, G * D).to(T)
    if case["mode"] != "train":
        return [y]
    gy, slope = s["grads"][0].float().view(R, G, D), sig * (1 + at * (1 - sig))
    gu = gy * slope if gate is None else gy * gate * sig
    gx = gu if w is None else gu * w
    gx = gx - xh * (gx * xh).mean(-1, keepdim=True) - (0 if case["rms"] else gx.mean(-1, keepdim=True))
    res = [y, (gx * rstd).view(R, G * D).to(T)]
    if w is not None:
        res.append((gu * xh).sum(0).flatten())
    if s["bias"] is not None:
        res.append(gu.sum(0).flatten())
    if gate is not None:
        res.append((gy * u * slope).view(R, G * D).to(T))
    return res


# ------------------------------------------------------------------ the framework's operators

def _own(s):
    fwp = importlib.import_module("recurrent-fwp_amd")
    case = s["case"]
    if case["op"] == "sum":
        return (fwp.decayed_sum(s["q"], s["k"], s["v"], s["decay"], s["W"], scale=s["scale"], lengths=s["lengths"]),)
    if case["op"] == "rotary":
        return fwp.rotary(s["q"], s["k"], s["frequencies"], positions=s["positions"], interleaved=case["interleaved"], scale=s["scale"],
                          lengths=s["lengths"])
    return (fwp.group_norm(s["x"], case["groups"], s["weight"], s["bias"], gate=s["gate"], eps=EPS, rms=case["rms"], activation="silu"),)


def run(state):
    s, case = state, state["case"]
    if not own:
        with torch.no_grad():
            return {"sum": _plain_sum, "rotary": _plain_rotary, "norm": _plain_norm}[case["op"]](s)
    if case["mode"] == "train":
        outs = _own(s)
        grads = torch.autograd.grad(outs, [s[k] for k in s["diff"]], s["grads"])
        return [o.detach() for o in outs] + list(grads)
    with torch.no_grad():
        outs = list(_own(s))
    return outs + ([s["W"]] if case["op"] == "sum" else [])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size, train = (4 if case["dtype"] == "fp32" else 2), case["mode"] == "train"
    if case["op"] == "norm":
        C = case["groups"] * case["size"]
        n, params = case["rows"] * C, 4 * C * (case["affine"] + (case["affine"] and not case["rms"]))
        b, f = n * size * (3 if case["gated"] else 2) + params, 14 * n
        if train:
            b, f = b + n * size * (3 if case["gated"] else 2) + params, f + 30 * n
        return {"bytes": b, "flops": f}
    N, H, G, L = (case[k] for k in ("N", "H", "G", "L"))
    if case["op"] == "rotary":
        n = N * L * (H + G)
        b, f = 2 * n * case["D"] * size + 4 * case["width"], 3 * n * case["width"]
        return {"bytes": 2 * b if train else b, "flops": 2 * f if train else f}
    E, M = case["E"], case["M"]
    rows = N * L * (2 * G * E + 2 * H * M) * size + 4 * H * (N * L if case["token_decay"] else 1)      # q, k, v, o and the decays
    b, f = rows, 4 * N * H * L * E * M
    if train:
        b, f = 2 * rows, 3 * f
    else:
        b += 2 * 4 * N * H * E * M
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ in 64 bits, from the definitions

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
    s = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    train = case["mode"] == "train"
    leaves = [s[k].requires_grad_() for k in s["diff"]] if train else []
    with torch.set_grad_enabled(train):
        outs = {"sum": _exact_sum, "rotary": _exact_rotary, "norm": _exact_norm}[case["op"]](s, case)
        if not train:
            return outs
        outs = outs[:len(s["grads"])]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [g.double() for g in s["grads"]]))


def _alive(s, case):
    n = torch.full((case["N"],), case["L"], device="cuda") if s["lengths"] is None else s["lengths"]
    return torch.arange(case["L"], device="cuda")[:, None] < n[None]                  # [L,N]


def _steps(W, q, k, v, g):
    """The recurrence over some steps: (the state behind them, what they read)."""
    outs = []
    for qt, kt, vt, gt in zip(q.unbind(0), k.unbind(0), v.unbind(0), g.unbind(0)):
        W = torch.exp(gt)[..., None, None] * W + kt[..., None] * vt[..., None, :]
        outs.append((qt[..., None] * W).sum(-2))
    return W, torch.stack(outs)


def _exact_sum(s, case):
    """The recurrence step by step; a backward pass goes through parts of 16 steps again."""
    N, H, G, L = (case[k] for k in ("N", "H", "G", "L"))
    alive = _alive(s, case)[:, :, None, None]
    first = lambda t: torch.where(alive, t.permute(2, 0, 1, 3), 0.0)                  # [L,N,heads,.], nothing in the rows behind a sequence
    per_head = lambda t: t[:, :, :, None].expand(L, N, G, H // G, t.shape[-1]).reshape(L, N, H, t.shape[-1])
    q, k, v = per_head(first(s["q"])) * s["scale"], per_head(first(s["k"])), first(s["v"])
    g = s["decay"]
    g = first((g[None, :, None] + torch.zeros(N, H, L, device="cuda", dtype=torch.float64) if g.dim() == 1 else g)[..., None])[..., 0]
    W = torch.zeros(N, H, case["E"], case["M"], device="cuda", dtype=torch.float64) if s["W"] is None else s["W"]
    outs = []
    for i in range(0, L, 16):
        part = [t[i:i + 16] for t in (q, k, v, g)]
        W, o = checkpoint(_steps, W, *part, use_reentrant=False) if torch.is_grad_enabled() else _steps(W, *part)
        outs.append(o)
    return [torch.cat(outs).permute(1, 2, 0, 3), W]


def _exact_rotary(s, case):
    """Pairs as complex numbers, times the one that an angle stands for."""
    w, alive = case["width"], _alive(s, case).t()[:, None, :, None]
    at = torch.arange(case["L"], device="cuda").expand(case["N"], case["L"])
    at = (at if s["positions"] is None else at + s["positions"][:, None])[:, None, :, None].double()
    turn = torch.polar(torch.full((), s["scale"], device="cuda", dtype=torch.float64), at * s["frequencies"].double())

    def turned(x):
        x = torch.where(alive, x, 0.0)
        head, rest = x[..., :w], x[..., w:]
        pairs = head.unflatten(-1, (w // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, w // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat([(y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2), rest], -1)
    return [turned(s["q"]), turned(s["k"])]


def _exact_norm(s, case):
    G, D = case["groups"], case["size"]
    x = s["x"].unflatten(-1, (G, D))
    x = (F.rms_norm if case["rms"] else F.layer_norm)(x, (D,), eps=EPS).flatten(-2)
    u = x if s["weight"] is None else x * s["weight"]
    u = u if s["bias"] is None else u + s["bias"]
    return [F.silu(u) if s["gate"] is None else u * F.silu(s["gate"])]
