"""The short causal convolution and the selective scan against their formulas in 64 bits: every width of state, lengths from one step on, padded
batches, views, states that go on, graphs and streams.

Tolerances count roundings of 2^-24 against the same formulas with every term positive.  Forward, a term of the scan passes at most four
roundings a step (its decay: the product with A, the exponential to one unit, the product with the state; the addition), sums of E terms, and
the softplus (its exponential's argument is off by |pre| log2(e) 2^-24, ten more follow); the errors of the decays' exponents add up to 10 / e of 2^-24, for x exp(-x) <= 1 / e.  Backward a term passes
the steps twice, and sums over channels (M), and for parameters over all steps.  Results of fewer bits are off by half a step of theirs more."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import scan_formulas as F

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(got, want, size, roundings, what, dtype):
    assert got.shape == want.shape and got.dtype is dtype, what
    tol = roundings * F.EPS32 * size + F.half_step(dtype) * want.abs() + F.smallest(dtype)
    off = float(((F.double(got) - want).abs() - tol).max())      # NaN is not <= 0
    assert off <= 0, f"{what}: {off:.3e} beyond a tolerance of up to {float(tol.max()):.3e}"


def randn(g, *shape):
    return torch.randn(*shape, generator=g)


def rows(g, dtype, N, H, L, D, layout):
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


CONV = [  # N, H, L, D, K, layout, ragged, carried
    (1, 1, 1, 1, 1, "plain", False, False), (2, 1, 1, 8, 4, "plain", False, True), (3, 2, 2, 12, 4, "plain", False, True),
    (2, 1, 3, 64, 8, "steps", False, True), (2, 3, 33, 20, 2, "steps", True, True), (1, 1, 32, 256, 4, "slice", False, False),
    (5, 1, 70, 7, 3, "slice", True, True), (4, 2, 31, 68, 5, "strided", True, False), (2, 1, 129, 260, 4, "plain", False, True),
    (2, 2, 40, 16, 6, "same", False, False), (4, 1, 200, 33, 7, "plain", True, True), (1, 8, 1100, 4, 4, "steps", False, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,L,D,K,layout,ragged,carried", CONV)
@pytest.mark.parametrize("silu,biased", [(True, True), (False, False)])
def test_conv(fwp, N, H, L, D, K, layout, ragged, carried, silu, biased, dtype):
    g = torch.Generator().manual_seed(N + 10 * L + D + K)
    x = rows(g, dtype, N, H, L, D, layout)
    w, b = randn(g, H, D, K).cuda(), randn(g, H, D).cuda() if biased else None
    state = randn(g, N, H, K - 1, D).to(dtype).cuda() if carried else None
    gy = rows(g, dtype, N, H, L, D, "steps")
    n = lengths_of(N, L, g) if ragged else None
    ref = [F.double(t) for t in (x, w, b, state)]
    args = dict(silu=silu, lengths=n, gy=F.double(gy))
    want, size = F.conv(*ref, **args), F.conv(*ref, **args, absolute=True)
    first = None if state is None else state.clone()
    leaves = [t for t in (x.detach().requires_grad_(), w.requires_grad_(), b.requires_grad_() if biased else None) if t is not None]
    y = fwp.causal_conv(leaves[0], w, b, state, silu=silu, lengths=n)
    grads = torch.autograd.grad(y, leaves, gy)
    # K products and the bias, then the sigmoid (twelve roundings and the exponential's argument) or nothing
    forward = K + 24
    check(y, want[0], size[0] * 1.1, forward, "y", dtype)
    if carried:
        assert torch.equal(F.double(state), want[1])
        with torch.no_grad():
            assert torch.equal(fwp.causal_conv(x, w, b, first, silu=silu, lengths=n), y) and torch.equal(first, state)
    check(grads[0], want[2], size[2], 3 * K + 32, "gx", dtype)
    check(grads[1], want[3], size[3], 3 * K + 32 + N * L, "gw", torch.float32)
    if biased:
        check(grads[2], want[4], size[4], 3 * K + 32 + N * L, "gb", torch.float32)


SCAN = [  # N, H, L, E, M, layout, ragged, carried, gated
    (1, 1, 1, 1, 1, "plain", False, False, True), (2, 1, 1, 16, 64, "plain", False, True, True), (3, 2, 2, 4, 65, "plain", False, True, False),
    (2, 2, 15, 16, 49, "steps", False, False, True), (3, 1, 16, 3, 128, "slice", True, True, True), (2, 3, 17, 5, 10, "slice", False, True, False),
    (4, 1, 33, 8, 70, "plain", True, True, True), (1, 1, 200, 16, 64, "steps", False, True, True), (5, 2, 131, 11, 49, "slice", True, False, False),
    (2, 1, 70, 32, 33, "strided", True, True, True), (2, 1, 41, 17, 64, "plain", False, False, True), (1, 2, 100, 64, 20, "steps", False, True, True),
    (3, 1, 24, 33, 66, "plain", True, True, False), (2, 1, 40, 16, 32, "same", False, False, True), (1, 1, 700, 2, 3, "plain", False, True, True),
    (3, 1, 513, 16, 5, "steps", True, True, True), (4, 1, 150, 64, 70, "slice", True, True, True), (2, 2, 61, 49, 64, "steps", False, True, False),
    (2, 1, 600, 8, 130, "plain", True, True, True),
]


def scan_inputs(g, dtype, N, H, L, E, M, layout, carried, gated):
    t = dict(Q=rows(g, dtype, N, H, L, E, layout), K=rows(g, dtype, N, H, L, E, layout), V=rows(g, dtype, N, H, L, M, layout),
             delta=(2 * rows(g, dtype, N, H, L, M, layout)), A=-torch.exp(randn(g, H, E, M)).cuda(), D=randn(g, H, M).cuda(),
             delta_bias=(randn(g, H, M) - 1).cuda())
    t["Z"] = rows(g, dtype, N, H, L, M, layout) if gated else None
    t["W"] = randn(g, N, H, E, M).cuda() if carried else None
    return t


def formulas(t, softplus, n, go=None, absolute=False):
    names = ("Q", "K", "V", "delta", "A", "W", "D", "Z", "delta_bias")
    return F.scan(*(F.double(t[k]) for k in names), softplus=softplus, lengths=n, go=None if go is None else F.double(go), absolute=absolute)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,L,E,M,layout,ragged,carried,gated", SCAN)
def test_scan(fwp, N, H, L, E, M, layout, ragged, carried, gated, dtype):
    g = torch.Generator().manual_seed(N + 7 * L + E + M)
    t = scan_inputs(g, dtype, N, H, L, E, M, layout, carried, gated)
    n = lengths_of(N, L, g) if ragged else None
    go = rows(g, dtype, N, H, L, M, "steps")
    want, size = formulas(t, True, n, go), formulas(t, True, n, go, absolute=True)
    names = [k for k in ("Q", "K", "V", "delta", "A", "D", "Z", "delta_bias") if t[k] is not None]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    first = None if t["W"] is None else t["W"].clone()
    out = fwp.selective_scan(**t, softplus=True, lengths=n)
    grads = dict(zip(names, torch.autograd.grad(out, [t[k] for k in names], go)))
    forward, back = 4 * L + E + 64, 8 * L + 2 * E + M + 128
    check(out, want[0], size[0], forward, "out", dtype)
    if carried:
        check(t["W"], want[1], size[1], forward, "W", torch.float32)
    for k, i, more, kind in (("Q", 2, 0, dtype), ("K", 3, 0, dtype), ("V", 4, 0, dtype), ("delta", 5, 0, dtype), ("A", 6, N * L, torch.float32),
                             ("D", 7, N * L, torch.float32), ("Z", 8, 0, dtype), ("delta_bias", 9, N * L, torch.float32)):
        if k in grads:
            check(grads[k], want[i], size[i], back + more, "gradient of " + k, kind)
    with torch.no_grad():       # nothing recorded: the same numbers, from the single-step kernel (another order of the sum over E) for one step
        t["W"] = first
        again = fwp.selective_scan(**t, softplus=True, lengths=n)
        if L > 1:
            assert torch.equal(again, out)
        check(again, want[0], size[0], forward, "out without recording", dtype)


@pytest.mark.parametrize("L", [1, 40, 260])
def test_scan_without_its_options(fwp, L):
    """No D, no bias, no gate, steps as they are given; zero and large steps."""
    g = torch.Generator().manual_seed(L)
    t = scan_inputs(g, torch.float32, 2, 2, L, 16, 40, "plain", False, False)
    t["delta"] = torch.rand(2, 2, L, 40, generator=g).cuda() * (torch.rand(2, 2, L, 40, generator=g) < 0.8).cuda()
    t["delta"][0, 0, L // 2] = 1e4      # forgets everything; A is not below -1e2
    t["D"] = t["delta_bias"] = None
    go = randn(g, 2, 2, L, 40).cuda()
    want, size = formulas(t, False, None, go), formulas(t, False, None, go, absolute=True)
    names = ["Q", "K", "V", "delta", "A"]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    out = fwp.selective_scan(t["Q"], t["K"], t["V"], t["delta"], t["A"])
    grads = torch.autograd.grad(out, [t[k] for k in names], go)
    check(out, want[0], size[0], 4 * L + 80, "out", torch.float32)
    for k, got, i in zip(names, grads, (2, 3, 4, 5, 6)):
        check(got, want[i], size[i], 10 * L + 300, "gradient of " + k, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_and_tokens_go_on_from_one_another(fwp, dtype):
    """Convolution, then scan: a padded prompt in one call against its parts and its tokens one by one, each with the state of what came before."""
    N, L, D, E, K = 3, 150, 72, 16, 4
    g = torch.Generator().manual_seed(3)
    x, qk = rows(g, dtype, N, 1, L, D, "steps"), rows(g, dtype, N, 1, L, 2 * E, "steps")
    delta, z = rows(g, dtype, N, 1, L, D, "steps"), rows(g, dtype, N, 1, L, D, "steps")
    w, b, A = randn(g, 1, D, K).cuda() / 2, randn(g, 1, D).cuda(), -torch.exp(randn(g, 1, E, D)).cuda()
    n = torch.tensor([L, 0, 97]).cuda()

    def part(first, last, state, W, n):
        s = slice(first, last)
        y = fwp.causal_conv(x[:, :, s], w, b, state, silu=True, lengths=n)
        return fwp.selective_scan(qk[:, :, s, :E], qk[:, :, s, E:], y, delta[:, :, s], A, W, Z=z[:, :, s], delta_bias=b, softplus=True, lengths=n)

    with torch.no_grad():
        state, W = torch.zeros(N, 1, K - 1, D, dtype=dtype).cuda(), torch.zeros(N, 1, E, D).cuda()
        whole = part(0, L, state, W, n)
        for cuts in ([0, 1, 2, 64, 90, 150], list(range(L + 1))):
            s2, W2 = torch.zeros_like(state), torch.zeros_like(W)
            outs = [part(a, c, s2, W2, (n - a)) for a, c in zip(cuts, cuts[1:])]
            assert torch.equal(s2, state)
            # the convolution's rows are the same numbers; the scan's sums are grouped otherwise
            want = F.double(whole)
            tol = 16 * L * F.EPS32 * 100 + 2 * F.half_step(dtype) * want.abs() + F.smallest(dtype)
            assert ((F.double(torch.cat(outs, 2)) - want).abs() <= tol).all()
            assert ((W2 - W).abs() <= 16 * L * F.EPS32 * 100).all()
            assert not torch.cat(outs, 2)[1].any() and not torch.cat(outs, 2)[2, :, 97:].any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_padded_rows_hold_stays_there(fwp, value):
    N, L, M, E, K = 4, 70, 36, 9, 4
    g = torch.Generator().manual_seed(5)
    n = torch.tensor([70, 0, 1, 33]).cuda()
    dead = ~F.alive(n, N, L).cuda()
    t = scan_inputs(g, torch.float32, N, 1, L, E, M, "steps", True, True)
    w, go = randn(g, 1, M, K).cuda(), randn(g, N, 1, L, M).cuda()
    results = []
    for fill in (0.0, value):
        u = {k: (x.masked_fill(dead, fill) if k in ("Q", "K", "V", "delta", "Z") else x.clone()).detach() for k, x in t.items()}
        names = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias"]
        state = randn(torch.Generator().manual_seed(1), N, 1, K - 1, M).cuda()
        for k in names:
            u[k].requires_grad_()
        x = w.clone().requires_grad_()
        y = fwp.causal_conv(u["V"], x, None, state, silu=True, lengths=n)
        out = fwp.selective_scan(**{**u, "V": y}, softplus=True, lengths=n)
        results.append([out, y, state, u["W"], *torch.autograd.grad(out, [u[k] for k in names] + [x], go.masked_fill(dead, fill))])
    for a, b in zip(*results):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_infinities_and_nan_go_where_they_belong(fwp):
    """A NaN among the rows of one sequence and channel reaches that channel from its step on, and no other sequence."""
    g = torch.Generator().manual_seed(6)
    t = scan_inputs(g, torch.float32, 3, 1, 60, 16, 70, "plain", False, False)
    x = t["V"].clone()
    x[1, 0, 20, 3] = float("nan")
    with torch.no_grad():
        a, b = (fwp.selective_scan(**{**t, "V": v}, softplus=True) for v in (t["V"], x))
        bad = torch.zeros_like(a, dtype=torch.bool)
        bad[1, 0, 20:, 3] = True
        assert torch.equal(torch.isnan(b), bad) and torch.equal(a[~bad], b[~bad])
        w = randn(g, 1, 70, 4).cuda()
        y = fwp.causal_conv(x, w)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[1, 0, 20:24, 3] = True
        assert torch.equal(torch.isnan(y), bad)
        # the activation's limits: silu is 0 and inf, its slope 0 and 1
        x = torch.tensor([float("-inf"), float("inf"), -200.0, 200.0]).view(1, 1, 4, 1).cuda()
        assert torch.equal(fwp.causal_conv(x, torch.ones(1, 1, 1).cuda(), silu=True).flatten()[[0, 1, 3]].cpu(), torch.tensor([0.0, float("inf"), 200.0]))
    x.requires_grad_()
    slope, = torch.autograd.grad(fwp.causal_conv(x, torch.ones(1, 1, 1).cuda(), silu=True).sum(), x)
    assert torch.equal(slope.flatten().cpu(), torch.tensor([0.0, 1.0, 0.0, 1.0]))


def test_infinite_values_without_a_skip(fwp):
    """No D is no term at all, not zero times the value."""
    t = {k: torch.rand(1, 1, 30, n, generator=torch.Generator().manual_seed(7)).cuda() + 0.1 for k, n in (("Q", 5), ("K", 5), ("V", 3), ("delta", 3))}
    t["V"][0, 0, 10, 1] = float("inf")
    out = fwp.selective_scan(**t, A=-torch.ones(1, 5, 3).cuda())
    want = torch.zeros(30, 3, dtype=torch.bool).cuda()
    want[10:, 1] = True
    assert torch.equal(torch.isposinf(out[0, 0]), want) and not torch.isnan(out).any()


@pytest.mark.parametrize("E,L", [(4, 1), (4, 300), (16, 300), (40, 700)])
def test_entries_that_forget_at_once(fwp, E, L):
    """A decay of minus infinity is exp(..) = 0 for every step that there is and changes nothing behind a sequence's end: the formula with -1e30, whose
    products with the steps (above 1e-3) are as far below the smallest exponent."""
    g = torch.Generator().manual_seed(E + L)
    t = scan_inputs(g, torch.float32, 3, 1, L, E, 20, "plain", True, True)
    forgets = (torch.rand(1, E, 20, generator=g) < 0.3).cuda()
    n = torch.tensor([L, L // 2, 0]).cuda()
    want, size = (formulas({**t, "A": t["A"].masked_fill(forgets, -1e30)}, True, n, absolute=a) for a in (False, True))
    W = t["W"].clone()
    t["A"] = t["A"].masked_fill(forgets, float("-inf"))
    with torch.no_grad():
        out = fwp.selective_scan(**t, softplus=True, lengths=n)
    check(out, want[0], size[0], 4 * L + E + 64, "out", torch.float32)
    check(t["W"], want[1], size[1], 4 * L + E + 64, "W", torch.float32)
    names = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias"]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    out = fwp.selective_scan(**{**t, "W": W}, softplus=True, lengths=n)
    grads = torch.autograd.grad(out, [t[k] for k in names], torch.ones_like(out))
    assert all(torch.isfinite(x).all() for x in grads) and not grads[4][forgets].any()


def test_growth_of_nothing(fwp):
    """Steps below zero make the state grow, here by exp(256) and more over a part of the sequence that is worked on by itself: a state of zero stays one."""
    g = torch.Generator().manual_seed(14)
    L, E, M = 2048, 4, 8
    t = scan_inputs(g, torch.float32, 1, 1, L, E, M, "plain", False, True)
    t["A"], t["delta_bias"], t["delta"] = -torch.ones(1, E, M).cuda(), None, torch.full((1, 1, L, M), -2.0).cuda()
    t["V"][:, :, :-5] = 0
    go = randn(g, 1, 1, L, M).cuda()
    go[:, :, 3:-5] = 0
    want, size = formulas(t, False, None, go), formulas(t, False, None, go, absolute=True)
    names = ["Q", "K", "V", "delta", "A", "D", "Z"]
    go[:, :, -5:] = 0       # whose gradient would grow without bound on the way back
    want = want[:2] + formulas(t, False, None, go)[2:]
    size = size[:2] + formulas(t, False, None, go, absolute=True)[2:]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    out = fwp.selective_scan(**t)
    check(out, want[0], size[0], 4 * 5 + E + 64, "out", torch.float32)      # five steps from the first value on
    for k, got, i in zip(names, torch.autograd.grad(out, [t[k] for k in names], go), range(2, 9)):
        check(got, want[i], size[i], 8 * 5 + 2 * E + M + 128, "gradient of " + k, torch.float32)


def test_any_of_the_gradients_alone(fwp):
    g = torch.Generator().manual_seed(15)
    t = scan_inputs(g, torch.float32, 2, 1, 50, 16, 40, "steps", False, True)
    t["w"], t["b"] = randn(g, 1, 40, 4).cuda(), randn(g, 1, 40).cuda()
    go = randn(g, 2, 1, 50, 40).cuda()
    names = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias", "w", "b"]

    def gradients(of):
        u = {k: x if x is None else x.detach().requires_grad_(k in of) for k, x in t.items()}
        w, b = u.pop("w"), u.pop("b")
        out = fwp.selective_scan(**{**u, "V": fwp.causal_conv(u["V"], w, b, silu=True)}, softplus=True)
        return torch.autograd.grad(out, [{**u, "w": w, "b": b}[k] for k in of], go)

    for k, want in zip(names, gradients(names)):
        assert torch.equal(gradients([k])[0], want), k


def test_rows_shared_by_heads(fwp):
    """One q and k for all heads, as views that repeat them: their gradients are the sums over the heads (two roundings)."""
    g = torch.Generator().manual_seed(16)
    t = scan_inputs(g, torch.float32, 2, 3, 60, 16, 30, "plain", False, True)
    q, k = randn(g, 2, 1, 60, 16).cuda().requires_grad_(), randn(g, 2, 1, 60, 16).cuda().requires_grad_()
    go = randn(g, 2, 3, 60, 30).cuda()
    each = [x.detach().repeat(1, 3, 1, 1).requires_grad_() for x in (q, k)]
    a = fwp.selective_scan(**{**t, "Q": q.expand(2, 3, 60, 16), "K": k.expand(2, 3, 60, 16)}, softplus=True)
    b = fwp.selective_scan(**{**t, "Q": each[0], "K": each[1]}, softplus=True)
    assert torch.equal(a, b)
    for got, want in zip(torch.autograd.grad(a, [q, k], go), torch.autograd.grad(b, each, go)):
        assert float(((got - want.sum(1, keepdim=True)).abs() - 4 * F.EPS32 * want.abs().sum(1, keepdim=True)).max()) <= 0


def test_in_inference_mode(fwp):
    g = torch.Generator().manual_seed(17)
    t = scan_inputs(g, torch.bfloat16, 2, 1, 30, 16, 64, "steps", True, True)
    w, state = randn(g, 1, 64, 4).cuda(), torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16).cuda()

    def block(u, state):
        v = fwp.causal_conv(u["V"], w, None, state, silu=True)
        out = fwp.selective_scan(**{**u, "V": v}, softplus=True)
        return [out, *(x for x in fwp.residual_norm(out, u["Z"], after=w[0, :, 0], before=w[0, :, 1]) if x is not None), u["W"], state]

    with torch.no_grad():
        want = block({**t, "W": t["W"].clone()}, state.clone())
    W0 = t["W"].clone()
    with torch.inference_mode():        # states made here and outside
        inside = block({**t, "W": t["W"].clone()}, state.clone())
        outside = block(t, state)
    for a, b, c in zip(want, inside, outside):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert not torch.equal(W0, t["W"])


def test_the_same_call_gives_the_same_bits(fwp):
    g = torch.Generator().manual_seed(8)
    t = scan_inputs(g, torch.bfloat16, 3, 1, 400, 16, 200, "steps", False, True)
    names = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias"]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    w, go = randn(g, 1, 200, 4).cuda().requires_grad_(), rows(g, torch.bfloat16, 3, 1, 400, 200, "steps")
    seen = []
    for _ in range(3):
        out = fwp.selective_scan(**{**t, "V": fwp.causal_conv(t["V"], w, silu=True)}, softplus=True)
        seen.append([out, *torch.autograd.grad(out, [t[k] for k in names] + [w], go)])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_parameters_shared_by_two_calls_and_rows_used_twice(fwp):
    g = torch.Generator().manual_seed(9)
    x, A = randn(g, 2, 1, 30, 16).cuda().requires_grad_(), (-torch.rand(1, 16, 16, generator=g)).cuda().requires_grad_()
    go = randn(g, 2, 1, 30, 16).cuda()
    out = fwp.selective_scan(x, x, x, x, A, softplus=True)
    gx, gA = torch.autograd.grad(out, [x, A], go)
    y, want = (F.scan(*[F.double(x)] * 4, F.double(A), softplus=True, go=F.double(go), absolute=a) for a in (False, True))
    check(gx, y[2] + y[3] + y[4] + y[5], want[2] + want[3] + want[4] + want[5], 8 * 30 + 200, "x", torch.float32)
    out = fwp.selective_scan(x, x, x, x, A, softplus=True) + fwp.selective_scan(x, x, x, x, A, softplus=True)
    assert torch.equal(torch.autograd.grad(out, A, go)[0], gA + gA)


def test_graphs_and_streams(fwp):
    """Two captured graphs of the whole block, replayed in turn with eager work between, and the block on a stream of its own."""
    N, L, D, E = 2, 300, 40, 16
    g = torch.Generator().manual_seed(11)
    w, A = randn(g, 1, D, 4).cuda(), -torch.exp(randn(g, 1, E, D)).cuda()

    def block(x, qk, W):
        y = fwp.causal_conv(x, w, silu=True)
        return fwp.selective_scan(qk[..., :E], qk[..., E:], y, x, A, W, Z=x, softplus=True)

    def inputs():
        return randn(g, N, 1, L, D).cuda(), randn(g, N, 1, L, 2 * E).cuda(), randn(g, N, 1, E, D).cuda()

    with torch.no_grad():
        sets, graphs = [inputs(), inputs()], []
        side = torch.cuda.Stream()
        for x, qk, W in sets:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                block(x, qk, W.clone())
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = block(x, qk, W)
            graphs.append((graph, out))
        for turn in range(4):
            for (graph, out), (x, qk, W) in zip(graphs, sets):
                fresh = inputs()
                for to, src in zip((x, qk, W), fresh):
                    to.copy_(src)
                W0 = fresh[2].clone()
                graph.replay()
                want = block(x, qk, W0)
                torch.cuda.synchronize()
                assert torch.equal(out, want) and torch.equal(W, W0), turn
        x, qk, W = inputs()
        want, W1 = block(x, qk, W.clone()), W.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = block(x, qk, W1)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)


def test_a_captured_training_step(fwp):
    """Forward and backward of the block in one graph, with buffers that the gradients go to."""
    N, L, D, E = 2, 200, 48, 16
    g = torch.Generator().manual_seed(12)
    x, qk, go = randn(g, N, 1, L, D).cuda(), randn(g, N, 1, L, 2 * E).cuda(), randn(g, N, 1, L, D).cuda()
    w, A = randn(g, 1, D, 4).cuda(), -torch.exp(randn(g, 1, E, D)).cuda()
    leaves = [t.requires_grad_() for t in (x, qk, w, A)]

    def step():
        y = fwp.causal_conv(x, w, silu=True)
        out = fwp.selective_scan(qk[..., :E], qk[..., E:], y, x, A, softplus=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for turn in range(3):
        with torch.no_grad():
            for t in (x, qk, go):
                t.copy_(randn(g, *t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(kept, step()):
            assert torch.equal(a, b), turn


def test_a_state_that_was_kept_for_a_backward_pass_may_not_be_overwritten(fwp):
    W = torch.randn(1, 1, 16, 8).cuda().requires_grad_()
    square = (W.detach().requires_grad_() * 1.0)
    kept = square * square
    x = torch.randn(1, 1, 4, 8).cuda()
    q = torch.randn(1, 1, 4, 16).cuda()
    with torch.no_grad():
        fwp.selective_scan(q, q, x, x, -torch.ones(1, 16, 8).cuda(), square.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


def test_gradients_are_not_differentiated_again(fwp):
    x = torch.randn(1, 1, 20, 8).cuda().requires_grad_()
    w = torch.randn(1, 8, 4).cuda()
    for out in (fwp.causal_conv(x, w), fwp.selective_scan(x, x, x, x, -torch.ones(1, 8, 8).cuda()), fwp.residual_norm(x, x)[0]):
        with pytest.raises(RuntimeError, match="differentiated again"):      # raised inside the autograd engine
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_far_offsets(fwp):
    """Views whose steps lie more than 2^31 elements apart in all."""
    N, L, M, E = 2, 40, 8, 4
    g = torch.Generator().manual_seed(13)
    wide = torch.empty(L, 60_000_000, dtype=torch.float16, device="cuda")      # 4.8 GB
    at = 59_999_000
    block = wide[:, at:at + N * (3 * M + 2 * E)].view(L, N, 1, 3 * M + 2 * E)
    block.copy_(randn(g, L, N, 1, 3 * M + 2 * E))
    v, delta, z, q, k = (t.permute(1, 2, 0, 3) for t in block.split([M, M, M, E, E], -1))
    w, A = randn(g, 1, M, 4).cuda(), -torch.rand(1, E, M, generator=g).cuda()
    with torch.no_grad():
        got = [fwp.causal_conv(v, w), fwp.selective_scan(q, k, v, delta, A, Z=z, softplus=True)]
        v, delta, z, q, k = (t.contiguous() for t in (v, delta, z, q, k))
        want = [fwp.causal_conv(v, w), fwp.selective_scan(q, k, v, delta, A, Z=z, softplus=True)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
