"""The decayed sum rule with a state, in calls that are cut into segments and have more workgroups than the GPU holds at once: some start when others of the same head have
ended, and the state of before the call has to be what all of them go on from.

The formulas are those of decay_formulas.py, on the GPU in 64 bits and in blocks of 64 steps.  Tolerances as in test_gpu_decay.py; the decays are slow, so that the first state counts
for every step: it is worth some sqrt(E) of a result, thousands of times the tolerance."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F

BLOCK = 64


def formulas(q, k, v, g, W, scale, lengths=None):
    """(out, the last state); all of H heads, differentiable"""
    N, H, L, _ = v.shape
    live = torch.ones(N, 1, L, 1, dtype=torch.bool, device=q.device) if lengths is None else (torch.arange(L, device=q.device) < lengths[:, None])[:, None, :, None]
    q, k, v, g = (torch.where(live, t, 0.0) for t in (q * scale, k, v, g[..., None]))
    outs = []
    for i in range(0, L, BLOCK):
        qi, ki, vi, gi = (t[:, :, i:i + BLOCK] for t in (q, k, v, g))
        b = gi[..., 0].cumsum(-1)
        below = torch.ones(b.shape[-1], b.shape[-1], dtype=torch.bool, device=b.device).tril()
        apart = torch.where(below, torch.exp(torch.where(below, b[..., :, None] - b[..., None, :], 0.0)), 0.0)
        outs.append(((qi @ ki.transpose(-1, -2).contiguous()) * apart) @ vi + torch.exp(b)[..., None] * (qi @ W))
        W = torch.exp(b[..., -1])[..., None, None] * W + ki.transpose(-1, -2).contiguous() @ (torch.exp(b[..., -1:] - b)[..., None] * vi)
    return torch.cat(outs, 2), W


def inputs(dtype, N, H, L, E, M, ragged):
    g = torch.Generator(device="cuda").manual_seed(L + E + M)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    t = dict(Q=rnd(N, H, L, E).to(dtype), K=rnd(N, H, L, E).to(dtype), V=rnd(N, H, L, M).to(dtype), log_decay=-torch.exp(rnd(N, H, L)) / L)
    W, go, n = 4 * rnd(N, H, E, M), rnd(N, H, L, M).to(dtype), None
    if ragged:      # most of them end within the first segment, a few later
        n = torch.randint(0, L // 8, (N,), generator=g, device="cuda")
        n[::5], n[1::7], n[3] = L, L // 2 + 1, 0
    return t, W, go, n


def within(got, want, sizes, roundings, what, dtype):
    few = dtype is not torch.float32
    tol = F.EPS32 * (roundings * sizes[0] + 16 * sizes[1]) + (2.0 ** -16 * sizes[0] if few else 0.0) + F.half_step(dtype) * want.abs() + F.smallest(dtype)
    assert got.shape == want.shape and got.dtype is dtype, what
    off = float(((got.detach().double() - want).abs() - tol).max())      # NaN is not <= 0
    assert off <= 0, f"{what}: {off:.3e} beyond a tolerance of up to {float(tol.max()):.3e}"


# by the plan of these calls three to six segments, 1.6 to 2.8 times the workgroups that the GPU holds
CALLS = [(torch.float16, 24, 12, 2048, 128, 64, False), (torch.float32, 24, 12, 2048, 128, 64, False), (torch.bfloat16, 24, 12, 4096, 128, 64, False),
         (torch.bfloat16, 91, 1, 1962, 64, 128, False), (torch.float16, 8, 20, 1024, 128, 128, False), (torch.float32, 8, 20, 1024, 127, 100, False),
         (torch.bfloat16, 9, 16, 4096, 128, 128, False), (torch.bfloat16, 32, 12, 8192, 32, 32, False),
         (torch.float16, 24, 12, 2048, 128, 64, True), (torch.bfloat16, 91, 1, 1962, 64, 128, True), (torch.float32, 24, 12, 700, 100, 64, True)]


@pytest.mark.parametrize("dtype,N,H,L,E,M,ragged", CALLS)
def test_a_prompt_goes_on_from_its_state(fwp, dtype, N, H, L, E, M, ragged):
    t, W, _, n = inputs(dtype, N, H, L, E, M, ragged)
    args = [x.double() for x in t.values()]
    want = formulas(*args, W.double(), 0.3, n)
    positive = [x.abs() for x in args[:3]]
    sizes = list(zip(*[formulas(*positive, d, W.double().abs(), 0.3, n) for d in (args[3], args[3] / 2)]))
    with torch.no_grad():
        out = fwp.decayed_sum(**t, W=W, scale=0.3, lengths=n)
    within(out, want[0], sizes[0], 2 * E + 192 + L // 8, "out", dtype)
    within(W, want[1], sizes[1], 2 * E + 192 + L // 8, "W", torch.float32)


@pytest.mark.parametrize("dtype,N,H,L,E,M,ragged", [(torch.float16, 8, 20, 1024, 128, 128, False), (torch.bfloat16, 8, 20, 2048, 128, 128, True),
                                                    (torch.float32, 24, 12, 700, 128, 64, False)])
def test_training_goes_on_from_a_state(fwp, dtype, N, H, L, E, M, ragged):
    t, W, go, n = inputs(dtype, N, H, L, E, M, ragged)

    def both(values, W, go):
        leaves = [x.clone().requires_grad_() for x in values]
        out, last = formulas(*leaves, W, 0.3, n)
        return out.detach(), last.detach(), *torch.autograd.grad(out, leaves, go)
    args = [x.double() for x in t.values()]
    want = both(args, W.double(), go.double())
    positive = [x.abs() for x in args[:3]]
    sizes = []
    for d in (args[3], args[3] / 2):
        s = list(both([*positive, d], W.double().abs(), go.double().abs()))
        # a decay's gradient: of all that the 64 steps from this one on read and wrote, and of what is read beyond them of what was written before
        rows = (positive[0] * s[2]).sum(-1) + (positive[1] * s[3]).sum(-1)
        far = torch.nn.functional.pad(s[5][..., 1:], (0, 1))
        ahead = lambda x: torch.nn.functional.pad(x, (0, 63)).unfold(2, 64, 1)
        s[5] = ahead(rows).sum(-1) + ahead(far).amax(-1)
        sizes.append(s)
    sizes = list(zip(*sizes))
    leaves = {k: x.requires_grad_() for k, x in t.items()}
    out = fwp.decayed_sum(**leaves, W=W, scale=0.3, lengths=n)
    grads = torch.autograd.grad(out, list(leaves.values()), go)
    forward, backward = 2 * E + 192 + L // 8, 4 * (E + M) + 512 + L // 4 + 1
    within(out, want[0], sizes[0], forward, "out", dtype)
    within(W, want[1], sizes[1], forward, "W", torch.float32)
    for i, name in enumerate(t):
        within(grads[i], want[2 + i], sizes[2 + i], backward, "gradient of " + name, torch.float32 if name == "log_decay" else dtype)


def test_a_captured_prompt_goes_on_from_its_state(fwp):
    """Replays go on from one another, and from what the program writes into the state between them"""
    t, W, _, _ = inputs(torch.bfloat16, 91, 1, 1962, 64, 128, False)
    first = W.clone()
    call = lambda: fwp.decayed_sum(**t, W=W, scale=0.3)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        want = []
        W.copy_(first)
        for _ in range(3):
            want.append((call().clone(), W.clone()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for start in (first, 2 * first):
            W.copy_(start)
            for i in range(3):
                graph.replay()
                torch.cuda.synchronize()
                if start is first:
                    assert torch.equal(out, want[i][0]) and torch.equal(W, want[i][1])
                else:
                    assert not torch.equal(out, want[i][0]) and torch.isfinite(W).all()
