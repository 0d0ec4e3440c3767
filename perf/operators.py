"""The operators of the selective state space block, as they are measured: the short causal convolution, the selective
scan, and the norms around a block with its gate, scale and residual addition.

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

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _conv(mode, N, H, L, D, K, dtype, silu=True, ragged=False, time_major=False):
    return dict(op="conv", mode=mode, N=N, H=H, L=L, D=D, K=K, dtype=dtype, silu=silu, ragged=ragged, time_major=time_major)


def _scan(mode, N, H, L, E, M, dtype, gated=True, ragged=False, time_major=False):
    return dict(op="scan", mode=mode, N=N, H=H, L=L, E=E, M=M, dtype=dtype, gated=gated, ragged=ragged, time_major=time_major)


def _norm(mode, rows, cols, dtype, rms=False, gate="none", wide_stream=False):
    return dict(op="norm", mode=mode, rows=rows, cols=cols, dtype=dtype, rms=rms, gate=gate, wide_stream=wide_stream)


def listed():
    return [
        # decoding: one token for each of 32 sequences of a model with d_model 256 (512 inner channels)
        dict(_conv("step", 32, 1, 1, 512, 4, "fp32"), name="conv_step"),
        # prompts of different lengths in one padded batch, a width that is no multiple of anything, a shorter filter
        dict(_conv("forward", 7, 1, 1531, 1001, 3, "fp16", ragged=True), name="conv_prompt_ragged"),
        # one layer of the language model's training step: 32 x 1024 tokens, tensors as a layer hands them over
        dict(_conv("train", 32, 1, 1024, 512, 4, "fp32", time_major=True), name="conv_train"),
        # decoding: the state of 32 sequences, 512 channels x 16
        dict(_scan("step", 32, 1, 1, 16, 512, "fp32"), name="scan_step"),
        # decoding for many users of a wider model: bound by the state's bytes
        dict(_scan("step", 256, 1, 1, 16, 2048, "bf16"), name="scan_step_many"),
        # one long prompt: few channels, all of the parallelism has to come from the sequence
        dict(_scan("forward", 1, 1, 8192, 16, 1024, "bf16"), name="scan_prompt"),
        # one layer of the language model's training step
        dict(_scan("train", 32, 1, 1024, 16, 512, "fp32", time_major=True), name="scan_train"),
        # groups of heads with odd sizes, a padded batch of 391 tokens, no gate
        dict(_scan("train", 30, 8, 391, 11, 49, "fp16", gated=False, ragged=True), name="scan_train_ragged"),
        # a wider model's training step on long sequences
        dict(_scan("train", 8, 1, 2048, 16, 2048, "bf16"), name="scan_train_wide"),
        # decoding: the norms between two blocks for 32 rows
        dict(_norm("forward", 32, 256, "fp32"), name="norm_step"),
        # one layer of the language model's training step, gated
        dict(_norm("train", 32768, 256, "fp32", gate="sigmoid"), name="norm_train"),
        # a wide model in bf16 with its residual stream in 32 bits
        dict(_norm("train", 16384, 4096, "bf16", rms=True, wide_stream=True), name="norm_train_wide"),
    ]


def _between(rng, lo, hi):
    """A whole number from [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("conv", "scan", "scan", "norm"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op == "norm":
        cols = _between(rng, 17, 8192)
        rows = _between(rng, 1, max(1, min(65536, (1 << 26) // cols)))
        return _norm(rng.choice(("train", "train", "forward")), rows, cols, dtype, rng.random() < 0.5,
                     rng.choice(("none", "sigmoid", "silu", "rows")), rng.random() < 0.4)
    mode = rng.choice(("train", "train", "forward", "step"))
    H = rng.choice((1, 1, 8))
    L = 1 if mode == "step" else _between(rng, 2, 8192)
    ragged, time_major = mode != "step" and rng.random() < 0.3, rng.random() < 0.5
    if op == "conv":
        D = _between(rng, 8, 4096 // H)
        N = _between(rng, 1, max(1, min(256, (1 << 25) // (L * H * D))))
        return _conv(mode, N, H, L, D, rng.choice((2, 3, 4, 4, 4, 5, 8)), dtype, rng.random() < 0.7, ragged, time_major)
    E = rng.choice((16, 16, 8, 32, 64, _between(rng, 1, 64)))
    M = _between(rng, 8, 4096 // H)
    L = min(L, max(1, (1 << 28) // (E * H * M)))
    N = _between(rng, 1, max(1, min(256, (1 << 28) // (L * H * E * M))))
    return _scan(mode, N, H, L, E, M, dtype, rng.random() < 0.7, ragged, time_major)


# ------------------------------------------------------------------ inputs

def _rows(g, case, width, dtype=None):
    """N(0,1) values [N,H,L,width], or the permuted view of [L,N,H,width] storage that a layer has."""
    N, H, L = case["N"], case["H"], case["L"]
    shape = (L, N, H, width) if case["time_major"] else (N, H, L, width)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype or TYPES[case["dtype"]])
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


def _prepare_conv(case, g):
    N, H, D, K = (case[k] for k in ("N", "H", "D", "K"))
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    s = dict(x=_rows(g, case, D), weight=normal(H, D, K) / math.sqrt(K), bias=0.1 * normal(H, D), lengths=_lengths(g, case))
    # a training step starts at the sequence's start, a prompt and a token go on from what came before
    s["state"] = None if case["mode"] == "train" else normal(N, H, K - 1, D).to(TYPES[case["dtype"]])
    s["diff"] = ["x", "weight", "bias"]
    s["grad"] = _rows(g, case, D) if case["mode"] == "train" else None
    return s


def _prepare_scan(case, g):
    N, H, E, M = (case[k] for k in ("N", "H", "E", "M"))
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    # q and k are parts of one projection's rows, as a layer has them
    qk = _rows(g, case, 2 * E + 16)
    s = dict(q=qk[..., 16:16 + E], k=qk[..., 16 + E:], v=_rows(g, case, M), lengths=_lengths(g, case))
    # step sizes spread from 0.001 to 0.1 by channel, moved by the token; decays of 1 .. E at step size 1
    dt = torch.exp(torch.empty(H, M, device="cuda").uniform_(math.log(1e-3), math.log(0.1), generator=g))
    s["delta"] = _rows(g, case, M)
    s["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
    s["A"] = -(torch.arange(1.0, E + 1, device="cuda")[None, :, None] * torch.exp(0.1 * normal(H, E, M)))
    s["D"] = 1 + 0.1 * normal(H, M)
    s["z"] = _rows(g, case, M) if case["gated"] else None
    s["W"] = None if case["mode"] == "train" else 0.5 * normal(N, H, E, M)
    s["diff"] = ["q", "k", "v", "delta", "A", "D", "delta_bias"] + (["z"] if case["gated"] else [])
    s["grad"] = _rows(g, case, M) if case["mode"] == "train" else None
    return s


def _prepare_norm(case, g):
    R, C, T = case["rows"], case["cols"], TYPES[case["dtype"]]
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    s = dict(y=(0.3 * normal(R, C) + 0.1).to(T), x=normal(R, C).to(torch.float32 if case["wide_stream"] else T))
    s["gate"] = None if case["gate"] == "none" else normal(R, 1 if case["gate"] == "rows" else C).to(T)
    s["scale"] = 0.1 + 0.02 * normal(C)
    for name in ("after", "before"):
        s[name + "_weight"] = 1 + 0.1 * normal(C)
        s[name + "_bias"] = None if case["rms"] else 0.1 * normal(C)
    s["diff"] = [k for k in ("y", "x", "gate", "scale", "after_weight", "after_bias", "before_weight", "before_bias") if s[k] is not None]
    s["grad_r"], s["grad_n"] = normal(R, C).to(s["x"].dtype), normal(R, C).to(T)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"conv": _prepare_conv, "scan": _prepare_scan, "norm": _prepare_norm}[case["op"]](case, g)
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


def _silu_grad(x):
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def _plain_conv(s):
    case, T = s["case"], s["x"].dtype
    N, H, L, D, K = (case[k] for k in ("N", "H", "L", "D", "K"))
    valid, w = _valid(s), s["weight"].transpose(1, 2)[:, :, None]                    # [H,K,1,D]
    before = torch.zeros(N, H, K - 1, D, device="cuda") if s["state"] is None else s["state"].float()
    xs = torch.cat([before, _masked(s["x"].float(), valid)], 2)
    taps = [xs[:, :, j:j + L] for j in range(K)]
    p = s["bias"][:, None] + sum(w[:, j] * taps[j] for j in range(K))
    y = _masked(p * torch.sigmoid(p) if case["silu"] else p, valid).to(T)
    if s["state"] is not None:
        at = torch.full((N,), L, device="cuda") if valid is None else s["lengths"]
        at = at[:, None, None, None] + torch.arange(K - 1, device="cuda")[:, None]
        s["state"].copy_(xs.gather(2, at.expand(N, H, K - 1, D)).to(T))
        return [y, s["state"]]
    d = _masked(s["grad"].float(), valid)
    d = d * _silu_grad(p) if case["silu"] else d
    after = F.pad(d, (0, 0, 0, K - 1))
    gx = sum(w[:, j] * after[:, :, K - 1 - j:K - 1 - j + L] for j in range(K))
    gw = torch.stack([(d * taps[j]).sum((0, 2)) for j in range(K)], -1)
    return [y, _masked(gx, valid).to(T), gw, d.sum((0, 2))]


def _scanned(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 2, by doubling: log2(L) products over everything; overwrites both."""
    reach = 1
    while reach < a.shape[2]:
        b[:, :, reach:] += a[:, :, reach:] * b[:, :, :-reach]
        a[:, :, reach:] = a[:, :, reach:] * a[:, :, :-reach]
        reach *= 2
    return b


def _plain_scan(s):
    case, T = s["case"], s["v"].dtype
    valid = _valid(s)
    q, k, v = (_masked(s[n].float(), valid) for n in ("q", "k", "v"))
    pre = _masked(s["delta"].float(), valid) + s["delta_bias"][:, None]
    dt = _masked(torch.log1p(torch.exp(-pre.abs())) + pre.clamp(min=0), valid)
    step, A = dt[..., None, :], s["A"][:, None]                                       # [N,H,L,1,M], [H,1,E,M]
    a = torch.exp(step * A)
    b = (dt * v)[..., None, :] * k[..., None]
    if s["W"] is not None:
        b[:, :, 0] += a[:, :, 0] * s["W"]
    h = _scanned(a.clone(), b)
    o = (h * q[..., None]).sum(-2) + s["D"][:, None] * v
    z = None if s["z"] is None else _masked(s["z"].float(), valid)
    out = _masked(o if z is None else o * z * torch.sigmoid(z), valid).to(T)
    if s["W"] is not None:
        s["W"].copy_(h[:, :, -1])
        return [out, s["W"]]
    go = _masked(s["grad"].float(), valid)
    dy = go if z is None else go * z * torch.sigmoid(z)
    a = torch.cat([a[:, :, 1:], torch.zeros_like(a[:, :, :1])], 2)                    # the decay after a step
    g = _scanned(a.flip(2), (dy[..., None, :] * q[..., None]).flip(2)).flip(2)
    gq, gk = (h * dy[..., None, :]).sum(-1), (g * (dt * v)[..., None, :]).sum(-1)
    read = (g * k[..., None]).sum(-2)
    gv = dt * read + s["D"][:, None] * dy
    g[:, :, 1:] *= torch.exp(step[:, :, 1:] * A) * h[:, :, :-1]                       # g a W_{t-1}; the first W is zero
    g[:, :, 0] = 0
    gdt = v * read + (g * A).sum(-2)
    gdelta = _masked(gdt * torch.sigmoid(pre), valid)
    grads = [gq.to(T), gk.to(T), gv.to(T), gdelta.to(T), (g * step).sum((0, 2)), (dy * v).sum((0, 2)), gdelta.sum((0, 2))]
    if z is not None:
        grads.append((go * o * _silu_grad(z)).to(T))
    return [out, *grads]


EPS = 1e-5


def _normal(x, rms):
    """(the rows normalised, 1 / their spread)"""
    x = x if rms else x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _normal_grad(g, xh, rstd, rms):
    g = g - xh * (g * xh).mean(-1, keepdim=True) - (0 if rms else g.mean(-1, keepdim=True))
    return g * rstd


def _plain_norm(s):
    case, rms = s["case"], s["case"]["rms"]
    y, x = s["y"].float(), s["x"].float()
    yh, y_rstd = _normal(y, rms)
    u = yh * s["after_weight"] if rms else yh * s["after_weight"] + s["after_bias"]
    gate = None if s["gate"] is None else s["gate"].float()
    act = 1.0 if gate is None else gate * torch.sigmoid(gate) if case["gate"] == "silu" else torch.sigmoid(gate)
    r = x + s["scale"] * act * u
    rh, r_rstd = _normal(r, rms)
    n = rh * s["before_weight"] if rms else rh * s["before_weight"] + s["before_bias"]
    res = [r.to(s["x"].dtype), n.to(s["y"].dtype)]
    if case["mode"] != "train":
        return res
    gn = s["grad_n"].float()
    dr = s["grad_r"].float() + _normal_grad(gn * s["before_weight"], rh, r_rstd, rms)
    du = dr * s["scale"] * act
    grads = [_normal_grad(du * s["after_weight"], yh, y_rstd, rms).to(s["y"].dtype), dr.to(s["x"].dtype)]
    if gate is not None:
        slope = _silu_grad(gate) if case["gate"] == "silu" else act * (1 - act)
        gg = dr * s["scale"] * u * slope
        grads.append((gg.sum(-1, keepdim=True) if case["gate"] == "rows" else gg).to(s["gate"].dtype))
    grads += [(dr * act * u).sum(0), (du * yh).sum(0)] + ([] if rms else [du.sum(0)])
    return res + grads + [(gn * rh).sum(0)] + ([] if rms else [gn.sum(0)])


# ------------------------------------------------------------------ the framework's operators

def _own(s):
    fwp = importlib.import_module("recurrent-fwp_amd")
    case = s["case"]
    if case["op"] == "conv":
        return (fwp.causal_conv(s["x"], s["weight"], s["bias"], s["state"], silu=case["silu"], lengths=s["lengths"]),)
    if case["op"] == "scan":
        return (fwp.selective_scan(s["q"], s["k"], s["v"], s["delta"], s["A"], s["W"], D=s["D"], Z=s["z"],
                                   delta_bias=s["delta_bias"], softplus=True, lengths=s["lengths"]),)
    return fwp.residual_norm(s["y"], s["x"], after=(s["after_weight"], s["after_bias"]), gate=s["gate"], scale=s["scale"],
                             before=(s["before_weight"], s["before_bias"]), eps=EPS, rms=case["rms"],
                             activation=None if s["gate"] is None else "silu" if case["gate"] == "silu" else "sigmoid")


def run(state):
    s, case = state, state["case"]
    if not own:
        with torch.no_grad():
            return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[case["op"]](s)
    if case["mode"] == "train":
        outs = _own(s)
        gouts = [s["grad_r"], s["grad_n"]] if case["op"] == "norm" else [s["grad"]]
        grads = torch.autograd.grad(outs, [s[k] for k in s["diff"]], gouts)
        return [o.detach() for o in outs] + list(grads)
    with torch.no_grad():
        outs = list(_own(s))
    kept = {"conv": "state", "scan": "W"}.get(case["op"])
    return outs + ([s[kept]] if kept else [])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size, train = (4 if case["dtype"] == "fp32" else 2), case["mode"] == "train"
    if case["op"] == "norm":
        n, wide = case["rows"] * case["cols"], 4 if case["wide_stream"] else size
        gate = {"none": 0, "rows": case["rows"] * size}.get(case["gate"], n * size)
        params = 4 * case["cols"] * (3 if case["rms"] else 5)
        b, f = 2 * n * size + 2 * n * wide + gate + params, 20 * n
        if train:
            b, f = b + 2 * n * size + 2 * n * wide + gate + params, f + 50 * n
        return {"bytes": b, "flops": f}
    rows = case["N"] * case["H"] * case["L"]
    if case["op"] == "conv":
        n, H, D, K = rows * case["D"], case["H"], case["D"], case["K"]
        b, f = 2 * n * size + 4 * H * D * (K + 1), 2 * n * (K + 4)
        if train:
            b, f = b + 2 * n * size + 4 * H * D * (K + 1), f + 2 * n * (2 * K + 4)
        else:
            b += 2 * case["N"] * H * (K - 1) * D * size
        return {"bytes": b, "flops": f}
    E, M, H = case["E"], case["M"], case["H"]
    inputs = 2 * E + (3 if case["gated"] else 2) * M
    b, f = rows * (inputs + M) * size + 4 * H * M * (E + 2), rows * M * (8 * E + 12)
    if train:
        b, f = b + rows * (inputs + M) * size + 4 * H * M * (E + 2), f + rows * M * (18 * E + 24)
    else:
        b += 2 * 4 * case["N"] * H * E * M
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ in 64 bits, from the definitions

def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
    s = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    train = case["mode"] == "train"
    leaves = [s[k].requires_grad_() for k in s["diff"]] if train else []
    with torch.set_grad_enabled(train):
        if case["op"] == "norm":
            outs, grads = _exact_norm(s, case), [s["grad_r"], s["grad_n"]]
        else:
            (out, state), grads = {"conv": _exact_conv, "scan": _exact_scan}[case["op"]](s, case), [s["grad"]]
            if not train:
                return [out, state]
            outs = [out]
        if not train:
            return outs
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads))


def _alive(s, case):
    n = torch.full((case["N"],), case["L"], device="cuda") if s["lengths"] is None else s["lengths"]
    return (torch.arange(case["L"], device="cuda")[:, None] < n[None]).double()       # [L,N]


def _exact_conv(s, case):
    N, H, L, D, K = (case[k] for k in ("N", "H", "L", "D", "K"))
    alive = _alive(s, case).t()[:, None, :, None]
    first = torch.zeros(N, H, K - 1, D, device="cuda", dtype=torch.float64) if s["state"] is None else s["state"]
    x = torch.cat([first, s["x"] * alive], 2).permute(0, 1, 3, 2).reshape(N, H * D, L + K - 1)
    # every window of K rows against the filter
    p = (x.unfold(-1, K, 1) * s["weight"].reshape(H * D, 1, K)).sum(-1) + s["bias"].reshape(-1, 1)
    y = (F.silu(p) if case["silu"] else p).view(N, H, D, L).transpose(2, 3) * alive
    if s["state"] is None:
        return y, None
    n = [L] * N if s["lengths"] is None else s["lengths"].tolist()
    rows = x.view(N, H, D, L + K - 1)
    return y, torch.stack([rows[i, :, :, n[i]:n[i] + K - 1].transpose(1, 2) for i in range(N)])


def _exact_scan(s, case):
    """The recurrence step by step."""
    alive = _alive(s, case)[:, :, None, None]                                         # [L,N,1,1]
    W = torch.zeros(case["N"], case["H"], case["E"], case["M"], device="cuda", dtype=torch.float64) if s["W"] is None else s["W"]
    D = s["D"]
    dts = (F.softplus(s["delta"] + s["delta_bias"][:, None], threshold=700).permute(2, 0, 1, 3) * alive).unbind(0)
    qs, ks, vs = (s[n].permute(2, 0, 1, 3).unbind(0) for n in ("q", "k", "v"))
    outs = []
    for q, k, v, dt in zip(qs, ks, vs, dts):
        W = torch.exp(dt[:, :, None] * s["A"]) * W + (dt * v)[:, :, None] * k[..., None]
        outs.append(torch.matmul(q[:, :, None], W)[:, :, 0] + D * v)
    o = torch.stack(outs)
    o = o if s["z"] is None else o * F.silu(s["z"]).permute(2, 0, 1, 3)
    return (o * alive).permute(1, 2, 0, 3), W


def _exact_norm(s, case):
    cols = (case["cols"],)
    norm = (lambda t, w, b: F.rms_norm(t, cols, w, EPS)) if case["rms"] else (lambda t, w, b: F.layer_norm(t, cols, w, b, EPS))
    u = s["scale"] * norm(s["y"], s["after_weight"], s["after_bias"])
    if s["gate"] is not None:
        u = u * (F.silu(s["gate"]) if case["gate"] == "silu" else torch.sigmoid(s["gate"]))
    r = s["x"] + u
    return [r, norm(r, s["before_weight"], s["before_bias"])]
