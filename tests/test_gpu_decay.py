"""The decayed sum rule, rotary positions and the norm of groups of channels against their formulas in 64 bits: every size of state, lengths from one step on, padded
batches, views, shared heads, states that go on, graphs and streams.

Tolerances count roundings of 2^-24 against the same formulas with every term positive.  Forward, a term of the sum passes a dot product over E keys, a sum over
the at most 64 steps of a chunk, two roundings at each of the chunks behind it (32 steps at least), and splits into parts that leave out 2^-24 each.  The error of an
exponent x is x 2^-24 of its exponential, and x exp(-x) <= 0.74 exp(-x / 2): a second size with half the decays counts it.  Backward, terms pass dot products over
M columns and E keys and the chunks on both sides.  Results of fewer bits than fp32 take parts that leave out 2^-16, and are off by half a step of
theirs more."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def randn(g, *shape):
    return torch.randn(*shape, generator=g)


def rows(g, dtype, N, H, L, D, layout="plain"):
    """[N,H,L,D] on the GPU in one of the memory orders a caller may have"""
    if layout == "plain":
        return randn(g, N, H, L, D).to(dtype).cuda()
    if layout == "steps":          # permuted view of [L,N,H,D]
        return randn(g, L, N, H, D).to(dtype).cuda().permute(1, 2, 0, 3)
    if layout == "slice":          # columns of a wider buffer, at an odd offset
        return randn(g, L, N, H, 2 * D + 3).to(dtype).cuda()[..., 3:3 + D].permute(1, 2, 0, 3)
    if layout == "strided":        # the last axis not contiguous
        return randn(g, N, H, D, L).to(dtype).cuda().transpose(2, 3)
    return randn(g, N, H, 1, D).to(dtype).cuda().expand(N, H, L, D)      # "same": one row for all steps


def lengths_of(N, L, g):
    n = torch.randint(1, L + 1, (N,), generator=g)
    n[0], n[-1] = 0, L + 5
    if N > 2:
        n[1] = 1
    if N > 3:
        n[2] = -2
    return n.cuda()


def decays(g, N, H, L, kind):
    if kind == "head":
        return -torch.exp(randn(g, H) - 3).cuda()
    d = -torch.exp(randn(g, N, H, L) - 2)
    if kind == "strong":           # some steps forget nearly all, some everything
        d[torch.rand(N, H, L, generator=g) < 0.1] = -40.0
        d[torch.rand(N, H, L, generator=g) < 0.05] = -float("inf")
    if kind == "turned":           # another memory order
        return d.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0)
    return d.cuda()


def check(got, want, sizes, roundings, what, dtype):
    """sizes: with the decays, and with half of them"""
    assert got.shape == want.shape and got.dtype is dtype, what
    few = dtype is not torch.float32
    tol = F.EPS32 * (roundings * sizes[0] + 16 * sizes[1]) + (2.0 ** -16 * sizes[0] if few else 0.0) + F.half_step(dtype) * want.abs() + F.smallest(dtype)
    off = float(((F.double(got) - want).abs() - tol).max())      # NaN is not <= 0
    assert off <= 0, f"{what}: {off:.3e} beyond a tolerance of up to {float(tol.max()):.3e}"


SUM = [  # N, H, heads of q, k, v, L, E, M, layout, ragged, carried, decay
    (1, 1, (1, 1, 1), 1, 1, 1, "plain", False, False, "token"), (2, 2, (2, 2, 2), 1, 16, 32, "plain", False, True, "head"),
    (2, 3, (3, 3, 3), 2, 8, 5, "plain", True, True, "token"), (3, 2, (2, 2, 2), 31, 32, 32, "steps", True, False, "head"),
    (2, 2, (1, 1, 2), 64, 33, 16, "plain", False, True, "strong"), (1, 4, (2, 4, 1), 65, 64, 64, "steps", False, False, "turned"),
    (4, 2, (2, 1, 2), 130, 48, 40, "slice", True, True, "token"), (2, 1, (1, 1, 1), 200, 64, 33, "plain", False, True, "strong"),
    (2, 2, (2, 2, 2), 96, 100, 128, "steps", False, True, "token"), (2, 6, (3, 2, 6), 77, 128, 64, "plain", True, False, "token"),
    (1, 2, (2, 2, 2), 150, 7, 70, "strided", False, True, "head"), (2, 1, (1, 1, 1), 70, 128, 129, "plain", True, True, "token"),
    (1, 2, (1, 2, 2), 90, 20, 300, "slice", False, False, "token"), (2, 2, (2, 2, 2), 40, 16, 16, "same", False, False, "head"),
    (1, 1, (1, 1, 1), 1100, 16, 16, "plain", False, True, "token"), (4, 1, (1, 1, 1), 700, 64, 20, "steps", True, True, "strong"),
    (1, 1, (1, 1, 1), 600, 128, 32, "plain", False, True, "head"),
]


def sum_inputs(g, dtype, N, H, G, L, E, M, layout, carried, decay):
    t = dict(Q=rows(g, dtype, N, G[0], L, E, layout), K=rows(g, dtype, N, G[1], L, E, layout), V=rows(g, dtype, N, G[2], L, M, layout),
             log_decay=decays(g, N, H, L, decay))
    return t, randn(g, N, H, E, M).cuda() if carried else None


def sum_formulas(t, W, scale, n, go=None, **more):
    d = {k: F.double(x) for k, x in t.items()}
    if "halved" in more:
        d["log_decay"] = d["log_decay"] / 2
        del more["halved"]
    return F.decayed_sum(d["Q"], d["K"], d["V"], d["log_decay"], F.double(W), scale, None if n is None else n.cpu(), F.double(go), **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,G,L,E,M,layout,ragged,carried,decay", SUM)
def test_decayed_sum(fwp, N, H, G, L, E, M, layout, ragged, carried, decay, dtype):
    g = torch.Generator().manual_seed(N + 7 * L + E + M)
    t, W = sum_inputs(g, dtype, N, H, G, L, E, M, layout, carried, decay)
    n = lengths_of(N, L, g) if ragged else None
    scale, go = 0.3, rows(g, dtype, N, H, L, M, "steps")
    want = sum_formulas(t, W, scale, n, go)
    sizes = [sum_formulas(t, W, scale, n, go, absolute=True), sum_formulas(t, W, scale, n, go, absolute=True, halved=True)]
    sizes = list(zip(*sizes))
    if n is not None:              # what lies behind a sequence is not read
        for name in ("Q", "K", "V"):
            dead = ~F.alive(n, N, L).cuda().expand_as(t[name])
            t[name] = torch.where(dead, float("nan") if name != "V" else float("inf"), t[name])
        if t["log_decay"].dim() == 3:
            t["log_decay"] = torch.where(~F.alive(n, N, L)[..., 0].cuda(), float("nan"), t["log_decay"])
        go = torch.where(F.alive(n, N, L).cuda(), go, float("nan"))
    leaves = {k: x.detach().requires_grad_() for k, x in t.items()}
    first = None if W is None else W.clone()
    out = fwp.decayed_sum(**leaves, W=W, scale=scale, lengths=n)
    grads = torch.autograd.grad(out, list(leaves.values()), go)
    forward = 2 * E + 192 + L // 8
    backward = 4 * (E + M) + 512 + L // 4
    check(out, want[0], sizes[0], forward, "out", dtype)
    if carried:
        check(W, want[1], sizes[1], forward, "W", torch.float32)
        if L > 1:      # a single step that saves nothing has a kernel of its own, which sums in another order
            with torch.no_grad():
                assert torch.equal(fwp.decayed_sum(**t, W=first, scale=scale, lengths=n), out) and torch.equal(first, W)
    heads = [H // x for x in G] + [1]
    for i, name in enumerate(["Q", "K", "V", "log_decay"]):
        extra = N * L if name == "log_decay" and t[name].dim() == 1 else heads[i]
        check(grads[i], want[2 + i], sizes[2 + i], backward + extra, "gradient of " + name, torch.float32 if i == 3 else dtype)


STEP = [(1, 1, (1, 1, 1), 1, 1), (3, 4, (4, 4, 4), 32, 32), (2, 6, (2, 3, 6), 41, 73), (5, 2, (1, 1, 2), 128, 64), (2, 2, (2, 2, 1), 16, 260),
        (3, 1, (1, 1, 1), 100, 6), (1, 3, (3, 3, 3), 128, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,G,E,M", STEP)
@pytest.mark.parametrize("carried", [True, False])
@pytest.mark.parametrize("decay", ["head", "strong"])
def test_single_steps(fwp, N, H, G, E, M, carried, decay, dtype):
    g = torch.Generator().manual_seed(N + E + M)
    n = torch.tensor([1, 0, 3, -1, 1][:N]).cuda() if N > 1 else None
    W = randn(g, N, H, E, M).cuda() if carried else None
    for _ in range(3 if carried else 1):
        t, _ = sum_inputs(g, dtype, N, H, G, 1, E, M, "plain", False, decay)
        want = sum_formulas(t, W, 0.5, n)
        sizes = list(zip(*(sum_formulas(t, W, 0.5, n, absolute=True, **x) for x in ({}, {"halved": True}))))
        kept = None if W is None else W.clone()
        with torch.no_grad():
            out = fwp.decayed_sum(**t, W=W, scale=0.5, lengths=n)
        check(out, want[0], sizes[0], E + 16, "out", dtype)
        if carried:
            check(W, want[1], sizes[1], 8, "W", torch.float32)
            if n is not None:
                assert torch.equal(W[1], kept[1])      # an empty row's state stays as it is


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cuts", [[0, 1, 2, 40, 64, 65, 200], [0, 130, 131, 132, 133, 200]])
def test_a_prompt_and_its_tokens_go_on_from_one_another(fwp, cuts, dtype):
    g = torch.Generator().manual_seed(3)
    t, W = sum_inputs(g, dtype, 2, 4, (2, 2, 4), 200, 48, 40, "steps", True, "token")
    want = sum_formulas(t, W, 1.0, None)
    sizes = list(zip(*(sum_formulas(t, W, 1.0, None, absolute=True, **x) for x in ({}, {"halved": True}))))
    parts = []
    with torch.no_grad():
        for a, b in zip(cuts, cuts[1:]):
            parts.append(fwp.decayed_sum(*(t[k][:, :, a:b] for k in ("Q", "K", "V", "log_decay")), W))
    # every call rounds the state once more
    check(torch.cat(parts, 2), want[0], sizes[0], 2 * 48 + 192 + 200, "out", dtype)
    check(W, want[1], sizes[1], 2 * 48 + 192 + 200, "W", torch.float32)


def test_long_prompts_are_cut_into_segments_that_join(fwp):
    """One head and 20000 steps, which many workgroups share, against the same steps 500 at a time"""
    g = torch.Generator().manual_seed(5)
    t, _ = sum_inputs(g, torch.float32, 1, 1, (1, 1, 1), 20000, 32, 32, "plain", False, "token")
    t["log_decay"] = t["log_decay"] * 0.01
    go = randn(g, 1, 1, 20000, 32).cuda()
    W, piecewise = torch.zeros(1, 1, 32, 32).cuda(), torch.zeros(1, 1, 32, 32).cuda()
    leaves = [x.requires_grad_() for x in t.values()]
    out = fwp.decayed_sum(*leaves, W)
    grads = torch.autograd.grad(out, leaves, go)
    with torch.no_grad():
        parts = [fwp.decayed_sum(*(x[:, :, i:i + 500] for x in leaves), piecewise) for i in range(0, 20000, 500)]
    assert float((torch.cat(parts, 2) - out).abs().max()) <= 1e-4 * float(out.abs().max())
    assert float((piecewise - W).abs().max()) <= 1e-4 * float(W.abs().max())
    # the gradients of the same call, in 64 bits on the last 300 steps: what the steps before them left is a state
    d = {k: F.double(x)[:, :, -300:] for k, x in t.items()}
    with torch.no_grad():
        before = torch.zeros(1, 1, 32, 32).cuda()
        fwp.decayed_sum(*(x[:, :, :-300].contiguous() for x in leaves), before)
    want = F.decayed_sum(d["Q"], d["K"], d["V"], d["log_decay"], F.double(before), 1.0, None, F.double(go)[:, :, -300:])
    for got, w in zip(grads, want[2:]):
        assert float((F.double(got)[:, :, -300:] - w).abs().max()) <= 1e-4 * float(w.abs().max())


def test_gradients_against_differences(fwp):
    g = torch.Generator().manual_seed(11)
    t, _ = sum_inputs(g, torch.float32, 2, 2, (1, 2, 2), 70, 20, 12, "plain", False, "token")
    go = randn(g, 2, 2, 70, 12).cuda()
    leaves = {k: x.requires_grad_() for k, x in t.items()}
    grads = torch.autograd.grad(fwp.decayed_sum(**leaves), list(leaves.values()), go)
    for (name, x), grad in zip(t.items(), grads):
        v, step = torch.randn(x.shape, generator=g, dtype=torch.float64), 1e-5
        at = {k: F.double(y) for k, y in t.items()}
        value = lambda s: (F.decayed_sum(*({**at, name: at[name] + s * v}).values())[0] * F.double(go)).sum()
        slope = float((value(step) - value(-step)) / (2 * step))
        mine = float((F.double(grad) * v).sum())
        # the difference is off by step^2 of the third derivative and 2^-53 / step of the value, the gradient by its roundings
        assert abs(slope - mine) <= 1e-4 * float(F.double(grad).norm()) * v.numel() ** 0.25 + 1e-4, name


def test_far_rows_and_offsets_beyond_32_bits(fwp):
    """Rows 2^25 elements apart, and sequences whose offset passes 2^31 elements"""
    g = torch.Generator().manual_seed(2)
    big = torch.zeros(3 << 30, dtype=torch.bfloat16, device="cuda")
    far = lambda sN, sL: big.as_strided((2, 1, 40, 16), (sN, 16, sL, 1))
    for sN, sL in (((1 << 31) + 64, 32), (64, 1 << 25)):
        q, k, v = (randn(g, 2, 1, 40, 16).to(torch.bfloat16).cuda() for _ in range(3))
        d = decays(g, 2, 1, 40, "token")
        view = far(sN, sL)
        view.copy_(k)
        with torch.no_grad():
            assert torch.equal(fwp.decayed_sum(q, view, v, d), fwp.decayed_sum(q, k, v, d))
            view.copy_(v)
            assert torch.equal(fwp.decayed_sum(q, k, view, d), fwp.decayed_sum(q, k, v, d))


# ------------------------------------------------------------------ rotary positions

ROTARY = [  # N, heads of q and k, L, D, pairs, layout, interleaved, positions, ragged
    (1, 1, 1, 1, 2, 1, "plain", False, None, False), (2, 4, 2, 33, 32, 16, "steps", False, "start", True), (2, 4, 2, 33, 32, 16, "steps", True, "each", False),
    (3, 2, 2, 1, 64, 10, "plain", False, "start", False), (2, 3, 1, 40, 37, 12, "slice", True, "start", False), (2, 3, 1, 40, 37, 9, "slice", False, "each", True),
    (1, 2, 0, 70, 96, 48, "plain", True, "start", False), (4, 8, 8, 5, 128, 32, "plain", False, "far", True), (1, 1, 1, 17, 9, 4, "strided", True, "far", False),
    (1, 16, 4, 300, 64, 32, "steps", True, None, False), (2, 2, 1, 50, 80, 20, "same", False, None, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,G,L,D,pairs,layout,interleaved,at,ragged", ROTARY)
def test_rotary(fwp, N, H, G, L, D, pairs, layout, interleaved, at, ragged, dtype):
    g = torch.Generator().manual_seed(N + L + D)
    x = [rows(g, dtype, N, h, L, D, layout) for h in (H, G) if h]
    f = F.frequencies(2 * pairs)
    p = {None: None, "start": torch.tensor([5, 100000, -3, 0])[:N], "each": torch.randint(-50, 1 << 20, (N, L), generator=g),
         "far": torch.tensor([(1 << 24) + 1, 1 << 30, 12345678, 1])[:N]}[at]
    n = lengths_of(N, L, g) if ragged else None
    scale = 1.25
    args = dict(positions=p, interleaved=interleaved, scale=scale, lengths=None if n is None else n.cpu())
    want = [F.rotary(F.double(t), f, **args) for t in x]
    if n is not None:
        x = [torch.where(F.alive(n, N, L).cuda(), t, float("nan")) for t in x]
    leaves = [t.detach().requires_grad_() for t in x]
    got = fwp.rotary(leaves[0], leaves[1] if G else None, f.cuda(), positions=None if p is None else p.cuda(), interleaved=interleaved, scale=scale,
                     lengths=n)
    assert (got[1] is None) == (not G)
    got = [t for t in got if t is not None]
    gos = [rows(g, dtype, N, t.shape[1], L, D, "steps") for t in x]
    grads = torch.autograd.grad(got, leaves, gos)

    def close(a, w, size, what):
        # sine and cosine (three roundings of their value at most one, and of the angle's rest), two products and a sum
        tol = 10 * F.EPS32 * size + F.half_step(dtype) * w.abs() + F.smallest(dtype)
        assert a.shape == w.shape and a.dtype is dtype and float(((F.double(a) - w).abs() - tol).max()) <= 0, what
    for i, t in enumerate(x):
        clean = torch.where(F.alive(n, N, L), F.double(t), 0.0)
        close(got[i], want[i], F.rotary(clean, f, **args, absolute=True), f"rows {i}")
        # the adjoint turns back
        ref = clean.clone().requires_grad_()
        back = torch.autograd.grad(F.rotary(ref, f, **args), ref, F.double(gos[i]))[0]
        close(grads[i], back, F.rotary(F.double(gos[i]), f, **args, absolute=True), f"gradient {i}")


def test_rotary_keeps_distances_and_frequencies_scale(fwp):
    f, s = fwp.rotary_frequencies(64)
    assert f.dtype is torch.float64 and s == 1.0 and torch.allclose(f, F.frequencies(64), rtol=1e-14)
    assert torch.allclose(fwp.rotary_frequencies(64, scaling="linear", factor=4)[0], f / 4, rtol=1e-14)
    slowed = fwp.rotary_frequencies(64, scaling="base", factor=4)[0]
    assert torch.allclose(slowed[-1], f[-1] / 4, rtol=1e-12) and slowed[0] == f[0]
    parts, s = fwp.rotary_frequencies(64, scaling="parts", factor=4, trained=2048)
    turns = F.turns_per(2048, f)
    assert torch.equal(parts[turns >= 32], f[turns >= 32]) and torch.allclose(parts[turns <= 1], f[turns <= 1] / 4, rtol=1e-14) and s > 1.1
    # queries and keys moved together keep their products
    g = torch.Generator().manual_seed(0)
    q, k = randn(g, 1, 1, 30, 64).cuda(), randn(g, 1, 1, 30, 64).cuda()
    with torch.no_grad():
        a = fwp.rotary(q, k, f.cuda())
        b = fwp.rotary(q, k, f.cuda(), positions=torch.tensor([1 << 20]).cuda())
    assert float((a[0] @ a[1].transpose(2, 3) - b[0] @ b[1].transpose(2, 3)).abs().max()) <= 64 * 40 * F.EPS32 * float(q.abs().max() * k.abs().max()) * 8


# ------------------------------------------------------------------ norm of groups

NORM = [(1, 1, 1), (7, 1, 16), (33, 8, 32), (100, 3, 125), (5, 40, 3), (9, 2, 1000), (64, 5, 64), (50, 16, 7), (300, 2, 513), (17, 33, 130), (2000, 4, 24)]


def norm_inputs(g, dtype, R, G, D, gated, affine, biased):
    C = G * D
    x, gate = (randn(g, R, C) + 0.2).to(dtype).cuda(), randn(g, R, C).to(dtype).cuda() if gated else None
    return x, (1 + 0.3 * randn(g, C)).cuda() if affine else None, (0.3 * randn(g, C)).cuda() if biased else None, gate


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,G,D", NORM)
@pytest.mark.parametrize("rms,gated,affine,biased,activation", [(False, True, True, True, "silu"), (True, False, True, False, "silu"),
                                                                  (False, False, False, True, None), (True, True, False, False, "sigmoid"),
                                                                  (False, True, True, False, None)])
def test_group_norm(fwp, R, G, D, rms, gated, affine, biased, activation, dtype):
    g = torch.Generator().manual_seed(R + G + D)
    x, w, b, gate = norm_inputs(g, dtype, R, G, D, gated, affine, biased)
    gy = randn(g, R, G * D).to(dtype).cuda()
    eps = 1e-3
    leaves = [t.requires_grad_() for t in (x, w, b, gate) if t is not None]
    y = fwp.group_norm(x, G, w, b, gate=gate, eps=eps, rms=rms, activation=activation)
    grads = torch.autograd.grad(y, leaves, gy)
    ref = [F.double(t).requires_grad_() for t in leaves]
    it = iter(ref)
    rx, rw, rb, rg = (None if t is None else next(it) for t in (x, w, b, gate))
    want = F.group_norm(rx, G, rw, rb, rg, eps, rms, activation)
    wants = torch.autograd.grad(want, ref, F.double(gy))

    # The rows normalised are off by (D + 8) roundings of the largest of the group over its spread; weight, bias, gate and activation bring a dozen more.
    # An activation's slope is at most 1.1, and moves by at most half of what its argument is off.
    with torch.no_grad():
        t = rx.unflatten(-1, (G, D))
        c = t if rms else t - t.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        off = (D + 20) * F.EPS32 * (t.abs().amax(-1, keepdim=True) * rstd + 1)
        wide = lambda v: v.expand(R, G, D).flatten(-2)
        big = lambda v: wide(v.unflatten(-1, (G, D)).abs().amax(-1, keepdim=True))
        weight = 1.0 if rw is None else rw.abs()
        u = (c * rstd).flatten(-2) * (1.0 if rw is None else rw) + (0.0 if rb is None else rb)
        act = F.act(rg, activation).abs() + 1 if gated else torch.ones_like(u)
        # the slope's own change with u counts where there is no gate
        tol_y = wide(off) * (weight + u.abs() + 1) * act * 1.2 + F.half_step(dtype) * want.abs() + F.smallest(dtype)
        assert y.dtype is dtype and float(((F.double(y) - want).abs() - tol_y).max()) <= 0
        gd = F.double(gy).abs()
        d = gd * act * 1.2 * weight * (1.0 if gated else 1.0)
        size = big(d) * (1 + big(c.flatten(-2)) * wide(rstd)) ** 2
        scale = {0: size * wide(rstd) * 8, 3: gd * (weight + u.abs() + 1) * 2}
        for i, (name, got, ref_grad) in enumerate(zip([k for k, t in zip(("x", "w", "b", "gate"), (x, w, b, gate)) if t is not None], grads, wants)):
            if name in ("x", "gate"):
                s = scale[0] if name == "x" else scale[3]
                tol = wide(off) * (1 + u.abs()) * s * 2 + F.half_step(dtype) * ref_grad.abs() + F.smallest(dtype)
                assert got.dtype is dtype
            else:      # sums over the rows
                tol = ((wide(off) + R * F.EPS32) * gd * act * 1.2 * (1 + big(c.flatten(-2)) * wide(rstd)) * (2 + u.abs()) * 2).sum(0)
                assert got.dtype is torch.float32
            assert got.shape == ref_grad.shape and float(((F.double(got) - ref_grad).abs() - tol).max()) <= 0, name


def test_group_norm_reads_rows_in_place(fwp):
    """Slices of wider rows, batch axes, permuted and expanded rows give what their copies give, gradients in the leaf's shape"""
    g = torch.Generator().manual_seed(4)
    buf = randn(g, 6, 5, 200).cuda()
    w, b = randn(g, 64).cuda(), randn(g, 64).cuda()
    for x, gate in ((buf[..., 3:67], buf[..., 70:134]), (buf.transpose(0, 1)[..., :64], buf[:5, :1, 100:164].expand(5, 6, 64)), (buf[2, 1, :64], buf[3, 1, 64:128]),
                    (buf[:, :1, :64], buf[:, 2:3, 1:65])):
        leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, gate)]
        y = fwp.group_norm(x, 4, w, b, gate=gate, activation="silu")
        z = fwp.group_norm(leaves[0].contiguous(), 4, w, b, gate=leaves[1].contiguous(), activation="silu")
        assert torch.equal(y, z)
        base = buf.clone().requires_grad_()
        v = base[..., 3:67]
        grad = torch.autograd.grad(fwp.group_norm(v, 4, w, b, activation="silu").sum(), base)[0]
        assert grad.shape == base.shape and float(grad[..., :3].abs().max()) == 0 and float(grad[..., 3:67].abs().max()) > 0


# ------------------------------------------------------------------ calls

def block(fwp, q, k, v, d, W, f, n, w, b, gate):
    """A run of the three as a layer has it"""
    L, N, H, M = gate.shape
    q, k = fwp.rotary(q, k, f, lengths=n)
    o = fwp.decayed_sum(q, k, v, d, W, scale=0.25, lengths=n).permute(2, 0, 1, 3).reshape(L, N, H * M)
    return fwp.group_norm(o, H, w, b, gate=gate.reshape(L, N, H * M), activation="silu")


def block_inputs(g, dtype, N=3, H=4, L=150, E=32, M=48):
    q, k, v = (rows(g, dtype, N, H, L, x, "steps") for x in (E, E, M))
    return [q, k, v, decays(g, N, H, L, "token"), None, F.frequencies(E).cuda(), lengths_of(N, L, g), randn(g, H * M).cuda(), randn(g, H * M).cuda(),
            randn(g, L, N, H, M).to(dtype).cuda()]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_run_of_them(fwp, dtype):
    g = torch.Generator().manual_seed(9)
    args = block_inputs(g, dtype)
    diff = [0, 1, 2, 3, 7, 8, 9]
    leaves = [args[i].detach().requires_grad_() for i in diff]
    for i, t in zip(diff, leaves):
        args[i] = t
    y = block(fwp, *args)
    gy = randn(g, *y.shape).to(dtype).cuda()
    grads = torch.autograd.grad(y, leaves, gy)
    ref = [F.double(t).requires_grad_() for t in leaves]
    n = args[6].cpu()
    q, k = (F.rotary(t, F.double(args[5]), lengths=n) for t in ref[:2])
    H, live = 4, F.alive(n, 3, 150)
    # the recurrence in a differentiable form: sums over all pairs of steps
    b = torch.where(live[..., 0], ref[3], 0.0).cumsum(-1)
    apart = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(torch.ones(150, 150, dtype=torch.bool).triu(1), -float("inf")))
    o = 0.25 * ((q @ k.transpose(2, 3)) * apart) @ torch.where(live, ref[2], 0.0)
    want = F.group_norm(torch.where(live, o, 0.0).permute(2, 0, 1, 3).reshape(150, 3, -1), H, ref[4], ref[5], ref[6].reshape(150, 3, -1), activation="silu")
    wants = torch.autograd.grad(want, ref, F.double(gy))
    # rows of bf16 round four times on the way (half a step, 2^-8, each), fp32 rows pass sums of 200 terms; an output's norm counts
    tol = 16 * 2.0 ** -8 if dtype is torch.bfloat16 else 2000 * F.EPS32
    for name, a, w in zip(["y"] + [str(i) for i in diff], [y, *grads], [want, *wants]):
        assert torch.isfinite(a).all() and float((F.double(a) - w).norm()) <= tol * float(w.norm()), name


def test_other_streams_and_graphs(fwp):
    """Captured once, replayed on new inputs with eager work between, against eager calls; two graphs that live at once"""
    g = torch.Generator().manual_seed(1)
    a, b = block_inputs(g, torch.bfloat16), block_inputs(g, torch.bfloat16)
    Ws = [randn(g, 3, 4, 32, 48).cuda() for _ in range(2)]
    side = torch.cuda.Stream()
    with torch.no_grad():
        want = []
        for t, W in zip((a, b), Ws):
            t[4] = W.clone()
            want.append((block(fwp, *t), t[4]))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            t = list(a)
            t[4] = Ws[0].clone()
            other = block(fwp, *t)
        side.synchronize()
        assert torch.equal(other, want[0][0]) and torch.equal(t[4], want[0][1])
        static = [x.clone() if torch.is_tensor(x) else x for x in a]
        static[4] = Ws[0].clone()
        graphs = []
        for _ in range(2):
            with torch.cuda.stream(side):
                block(fwp, *static)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = block(fwp, *static)
            graphs.append((graph, out))
        for i in range(4):
            src, W = ((a, b)[i % 2], Ws[i % 2])
            for s, x in zip(static, src):
                if torch.is_tensor(s):
                    s.copy_(x)
            static[4].copy_(W)
            graph, out = graphs[i // 2]
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i % 2][0]) and torch.equal(static[4], want[i % 2][1]), i
            block(fwp, *[x.clone() if torch.is_tensor(x) else x for x in b])      # eager work in between
            torch.cuda.synchronize()


def test_a_captured_training_step(fwp):
    g = torch.Generator().manual_seed(6)
    args = block_inputs(g, torch.float32)
    diff = [0, 1, 2, 3, 7, 8, 9]
    static = [x.detach().clone() if torch.is_tensor(x) else x for x in args]
    gy = randn(g, 150, 3, 4 * 48).cuda()

    def step(t):
        leaves = [t[i].detach().requires_grad_() for i in diff]
        t = list(t)
        for i, x in zip(diff, leaves):
            t[i] = x
        return torch.autograd.grad(block(fwp, *t), leaves, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(static)
    for seed in (1, 2, 3):
        fresh = block_inputs(torch.Generator().manual_seed(seed), torch.float32)
        for s, x in zip(static, fresh):
            if torch.is_tensor(s):
                s.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, step(fresh)):
            assert torch.equal(a, b)


def test_gradients_once_and_only_where_wanted(fwp):
    g = torch.Generator().manual_seed(8)
    t, _ = sum_inputs(g, torch.float32, 1, 2, (2, 2, 2), 20, 8, 8, "plain", False, "head")
    q = t["Q"].requires_grad_()
    out = fwp.decayed_sum(q, t["K"], t["V"], t["log_decay"])
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
    a, b = fwp.rotary(q, t["K"], F.frequencies(8).cuda())
    assert torch.autograd.grad(a.sum(), q)[0].shape == q.shape and b.requires_grad
    k = t["K"].requires_grad_()
    a, b = fwp.rotary(q.detach(), k, F.frequencies(8).cuda())
    assert torch.autograd.grad(b.sum(), k)[0].shape == k.shape
    # a state is of another version once it has gone on
    W = torch.zeros(1, 2, 8, 8).cuda()
    y = (W * q.sum()).sum()
    fwp.decayed_sum(q, t["K"], t["V"], t["log_decay"], W)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
