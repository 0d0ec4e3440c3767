"""The norms around a block with its gate, scale and residual addition against the formula in 64 bits, whose gradients are autograd's.

Tolerances: an element passes fewer than 128 roundings of 2^-24 (sums over a row are trees of at most 3 x 4 x 16 + 8 additions, two or
three of them in a row's gradient; sigmoid, square root and division a dozen), each against its terms with absolute values; sums over the rows as many as
there are rows more.  Results of fewer bits are off by half a step of theirs more."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import scan_formulas as F

CASES = [  # shape, rms, gate (None, "full", "one"), activation, scale, after (0: none, 1: weight, 2: with bias), before
    ((1, 1), False, None, None, False, 2, 2), ((1, 4), True, "full", "silu", True, 1, 1), ((3, 5), False, "one", "sigmoid", True, 2, 2),
    ((7, 64), False, "full", "sigmoid", True, 2, 2), ((5, 3, 100), True, "full", None, True, 1, 1), ((2, 255), False, "one", "silu", False, 2, 1),
    ((33, 256), False, "full", "silu", True, 2, 2), ((9, 257), True, None, None, True, 1, 1), ((6, 512), False, "full", "sigmoid", True, 0, 2),
    ((5, 640), True, "one", None, True, 1, 1), ((4, 1024), False, "full", "sigmoid", True, 2, 0), ((3, 1027), False, "full", "silu", True, 2, 2),
    ((3, 2048), True, None, None, True, 1, 1), ((2, 2050), False, "one", "sigmoid", True, 2, 2), ((3, 4096), True, "full", "silu", False, 1, 1),
    ((2, 4099), False, "full", None, True, 2, 2), ((2, 8192), False, "full", "sigmoid", True, 2, 2), ((3, 8191), True, "one", "silu", True, 1, 1),
    ((2100, 256), False, "full", "sigmoid", True, 2, 2), ((700, 1100), True, "one", "sigmoid", True, 1, 1), ((4, 96), False, None, None, False, 0, 0),
]
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.float32)]


def bound(size, want, dtype, more=0):
    return (128 + more) * F.EPS32 * size + F.half_step(dtype) * want.abs() + F.smallest(dtype)


def check(got, want, size, dtype, what, more=0):
    assert got.shape == want.shape and got.dtype is dtype, what
    off = (F.double(got) - want).abs() - bound(size, want, dtype, more)
    assert torch.isfinite(got).all() and float(off.max()) <= 0, (what, float(off.max()))


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("shape,rms,gating,act,scaled,after,before", CASES)
def test_rows(fwp, shape, rms, gating, act, scaled, after, before, dtype, stream):
    g = torch.Generator().manual_seed(sum(shape))
    cols, rows = shape[-1], 1
    for n in shape[:-1]:
        rows *= n
    randn = lambda *s: torch.randn(*s, generator=g)
    y, x = (randn(*shape) + 0.2).to(dtype).cuda(), (2 * randn(*shape)).to(stream).cuda()
    gate = None if gating is None else randn(*(shape if gating == "full" else (*shape[:-1], 1))).to(dtype).cuda()
    scale = (0.5 * randn(cols)).cuda() if scaled else None
    param = lambda n: [None, None] if n == 0 else [(1 + 0.2 * randn(cols)).cuda(), (0.3 * randn(cols)).cuda() if n == 2 else None]
    (aw, ab), (bw, bb) = param(after), param(before)
    gr, gn = randn(*shape).to(stream).cuda(), randn(*shape).to(dtype).cuda()

    # the reference, with a copy of each parameter for every row so that the rows' shares can be told apart
    each = lambda t: None if t is None else F.double(t).expand(rows, cols).clone().requires_grad_()
    flat = lambda t: None if t is None else F.double(t).reshape(rows, -1).requires_grad_()
    d = dict(y=flat(y), x=flat(x), aw=each(aw), ab=each(ab), gate=flat(gate), scale=each(scale), bw=each(bw), bb=each(bb))
    r, n = F.residual_norm(**d, eps=1e-5, rms=rms, act=act)
    leaves = {k: t for k, t in d.items() if t is not None}
    outs, gouts = ([r, n], [flat(gr).detach(), flat(gn).detach()]) if n is not None else ([r], [flat(gr).detach()])
    want = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gouts)))

    # absolute sizes of what is added up
    with torch.no_grad():
        def normal(t):
            t = t if rms else t - t.mean(-1, keepdim=True)
            s = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5)
            return (t * s).abs(), s
        one = torch.ones(rows, cols, dtype=torch.float64)
        yh, ys = normal(d["y"]) if after else (d["y"].abs(), 1.0)
        sc, act_v = one if scale is None else d["scale"].abs(), one if gate is None else F.activation(d["gate"], act).abs() * one
        slope = torch.zeros(1) if gate is None else torch.ones(1) if act is None else torch.full((1,), 1.1)
        awa, bwa = one if aw is None else d["aw"].abs(), one if bw is None else d["bw"].abs()
        big = lambda t: t + t.mean(-1, keepdim=True) + t.abs().max(-1, keepdim=True)[0] * 1e-2
        u = big(yh) * awa + (0 if ab is None else d["ab"].abs())
        r_size = d["x"].abs() + sc * act_v * u
        rh, rs = normal(r)
        n_size = big(big(r_size) * rs) * bwa + (0 if bb is None else d["bb"].abs())
        base = gouts[0].abs()
        if before:
            h = gouts[1].abs() * bwa
            rh = big(r_size) * rs
            base = base + rs * (h + h.mean(-1, keepdim=True) + rh * (h * rh).mean(-1, keepdim=True))
        du = base * sc * act_v
        h = du * awa
        gy = ys * (h + h.mean(-1, keepdim=True) + yh * (h * yh).mean(-1, keepdim=True)) if after else h
        sizes = dict(y=gy, x=base, gate=base * sc * u * slope, scale=base * act_v * u, aw=du * big(yh), ab=du)
        if before:
            sizes.update(bw=gouts[1].abs() * rh, bb=gouts[1].abs())

    got_leaves = {k: t.requires_grad_() for k, t in dict(y=y, x=x, aw=aw, ab=ab, gate=gate, scale=scale, bw=bw, bb=bb).items() if t is not None}
    got_r, got_n = fwp.residual_norm(y, x, after=(aw, ab), gate=gate, scale=scale, before=(bw, bb) if before == 2 else bw, rms=rms, activation=act)
    check(got_r.reshape(rows, cols), r.detach(), r_size, stream, "r")
    got_outs = [got_r]
    if n is None:
        assert got_n is None
    else:
        check(got_n.reshape(rows, cols), n.detach(), n_size, dtype, "n")
        got_outs.append(got_n)
    grads = dict(zip(got_leaves, torch.autograd.grad(got_outs, list(got_leaves.values()), [gr, gn][:len(got_outs)])))
    for k in ("y", "x"):
        check(grads[k].reshape(rows, cols), want[k], sizes[k], dtype if k == "y" else stream, "gradient of " + k)
    if gate is not None:
        size = sizes["gate"] if gating == "full" else sizes["gate"].sum(-1, keepdim=True)
        check(grads["gate"].reshape(rows, -1), want["gate"], size, dtype, "gradient of the gate")
    for k in ("scale", "aw", "ab", "bw", "bb"):
        if k in grads:
            check(grads[k], want[k].sum(0), sizes[k].sum(0), torch.float32, "gradient of " + k, rows)


def test_only_one_of_the_results_is_used(fwp):
    g = torch.Generator().manual_seed(0)
    y, x = (torch.randn(5, 300, generator=g).cuda().requires_grad_() for _ in range(2))
    w = torch.ones(300).cuda()
    zero = torch.zeros(5, 300).cuda()
    go = torch.randn(5, 300, generator=g).cuda()
    for i in (0, 1):
        one = torch.autograd.grad(fwp.residual_norm(y, x, after=w, before=w)[i], [y, x], go)
        both = torch.autograd.grad(fwp.residual_norm(y, x, after=w, before=w), [y, x], [go, zero] if i == 0 else [zero, go])
        assert all(torch.equal(a, b) for a, b in zip(one, both))


def test_rows_that_are_not_contiguous_or_aligned(fwp):
    """Views are the same call as their copies.  Rows and parameters at four bytes from a boundary are
    read by other loads: each result is within the 128 roundings of its terms, so two of them are within twice that of one another.  The terms of n are at most
    8 here (r below 16 times the spread), those of r 32."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(40, 6, 130, generator=g).cuda()
    y, x, w = wide[:, ::2, 2:130], wide.transpose(0, 1)[:3, :, 2:].permute(1, 0, 2), torch.randn(128, generator=g).cuda()
    views = fwp.residual_norm(y, x, after=(w, w), before=(w, w), scale=w)
    plain = fwp.residual_norm(y.contiguous(), x.contiguous(), after=(w, w), before=(w, w), scale=w)
    for a, b in zip(views, plain):
        assert torch.equal(a, b)
    shifted = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    for args in ((shifted(y.contiguous()), x, w), (y, x, shifted(w))):
        odd = fwp.residual_norm(args[0], args[1], after=(args[2], w), before=(w, args[2]), scale=w)
        for a, b, size in zip(odd, plain, (32.0, 32.0)):
            assert float((a - b).abs().max()) <= 2 * 128 * F.EPS32 * size


def test_constant_rows_and_large_means(fwp):
    """A row without spread is divided by sqrt(eps); one far from zero keeps what its elements can tell apart."""
    y = torch.full((2, 512), 7.0).cuda()
    x = torch.zeros(2, 512).cuda()
    w = torch.ones(512).cuda()
    r, n = fwp.residual_norm(y, x, after=w, before=w)
    assert not r.any() and not n.any()
    y = (4096 + torch.randint(-8, 9, (3, 512), generator=torch.Generator().manual_seed(2))).float().cuda()      # exact sums
    r, _ = fwp.residual_norm(y, torch.zeros(3, 512).cuda(), after=w)
    want = F.residual_norm(F.double(y), torch.zeros(3, 512, dtype=torch.float64), F.double(w))[0]
    assert float((F.double(r) - want).abs().max()) <= (4096 + 64) * F.EPS32      # the mean is off by a rounding of 4096, the spread is about 5


def test_parameters_gradients_are_tensors_of_their_own(fwp):
    """They share memory, not a byte of it: accumulated, cleared and changed one by one."""
    g = torch.Generator().manual_seed(6)
    y, x = torch.randn(9, 131, generator=g).cuda(), torch.randn(9, 131, generator=g).cuda()
    params = [torch.randn(131, generator=g).cuda().requires_grad_() for _ in range(5)]

    def backward():
        r, n = fwp.residual_norm(y, x, after=(params[0], params[1]), scale=params[2], before=(params[3], params[4]))
        (r * x + n * y).sum().backward()

    backward()
    once = [p.grad.clone() for p in params]
    backward()
    for p, a in zip(params, once):
        assert p.grad.is_contiguous() and torch.equal(p.grad, a + a)
    for i, p in enumerate(params):
        p.grad.fill_(float(i))
    assert all(bool((p.grad == float(i)).all()) for i, p in enumerate(params))


def test_infinite_rows_that_a_gate_masks(fwp):
    """Without a norm on y the gradients do not pass y's values: where an infinite one is masked away by the caller, gy is as for any other."""
    g = torch.Generator().manual_seed(4)
    y, x, gate, gr = (torch.randn(6, 300, generator=g).cuda() for _ in range(4))
    scale = torch.randn(300, generator=g).cuda()
    masked = torch.zeros(6, 300, dtype=torch.bool).cuda()
    masked[1, 7] = masked[4, 299] = masked[5, 0] = True
    gr = gr.masked_fill(masked, 0)
    seen = []
    for fill in (0.0, float("inf"), float("nan")):
        leaves = [y.masked_fill(masked, fill).requires_grad_(), x.clone().requires_grad_()]
        r, _ = fwp.residual_norm(leaves[0], leaves[1], gate=gate, scale=scale, activation="sigmoid")
        seen.append(torch.autograd.grad(r, leaves, gr))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))
    assert torch.equal(seen[0][1], gr)


def test_more_than_two_to_the_31_elements(fwp):
    """The last rows of a tensor whose offsets pass 32 bits are as those of a small one."""
    rows, cols = (1 << 18) + 5, 8192
    g = torch.Generator().manual_seed(5)
    few = [torch.randn(4, cols, generator=g).to(torch.bfloat16).cuda() for _ in range(4)]
    w = torch.randn(cols, generator=g).cuda()
    y, x, gr, gn = (torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    for big, small in zip((y, x, gr, gn), few):
        big[:2], big[-2:] = small[:2], small[2:]
    results = []
    for y_, x_, gr_, gn_ in ((y, x, gr, gn), few):
        y_, x_ = y_.requires_grad_(), x_.requires_grad_()
        r, n = fwp.residual_norm(y_, x_, after=w, before=w, rms=True)
        results.append([r.detach(), n.detach(), *torch.autograd.grad([r, n], [y_, x_], [gr_, gn_])])
    for a, b in zip(*results):
        assert torch.equal(a[:2], b[:2]) and torch.equal(a[-2:], b[2:])


def test_a_captured_step_beside_eager_work(fwp):
    g = torch.Generator().manual_seed(3)
    y, x, gate = (torch.randn(50, 1200, generator=g).cuda() for _ in range(3))
    w = torch.randn(1200, generator=g).cuda().requires_grad_()
    gr = torch.randn(50, 1200, generator=g).cuda()

    def step():
        r, n = fwp.residual_norm(y, x, after=w, gate=gate, scale=w, before=w, activation="silu")
        return [r.detach(), n.detach(), *torch.autograd.grad([r, n], w, [gr, gr])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for _ in range(3):
        for t in (y, x, gate):
            t.copy_(torch.randn(50, 1200, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
