"""The decayed sum rule with so many heads that a kernel with a workgroup for every 64 numbers of every state would be beyond a launch.  Tolerances as in test_gpu_decay.py: a
result has at most 2 E + 192 roundings of its terms, a gradient 4 (E + M) + 512, and those of 16 bits leave out 2^-16."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F


def within(got, want, size, roundings, what):
    tol = (F.EPS32 * (roundings + 16) + 2.0 ** -16) * size + F.half_step(torch.bfloat16) * want.abs() + F.smallest(torch.bfloat16)
    assert got.shape == want.shape and float(((got.detach().double() - want).abs() - tol).max()) <= 0, what


@pytest.mark.parametrize("N,H,E", [(4096, 8, 128), (1 << 17, 1, 64)])
def test_two_steps_of_many_heads(fwp, N, H, E):
    g = torch.Generator(device="cuda").manual_seed(E)
    q, k, v = (torch.randn(N, H, 2, E, generator=g, device="cuda").bfloat16() for _ in range(3))
    d = torch.linspace(-2, -0.1, H, device="cuda")
    with torch.no_grad():
        out = fwp.decayed_sum(q, k, v, d, scale=0.3)

    def formula(q, k, v):
        dot = lambda s, t: (q[:, :, s] * k[:, :, t]).sum(-1, keepdim=True) * 0.3
        first = dot(0, 0) * v[:, :, 0]
        return torch.stack([first, dot(1, 1) * v[:, :, 1] + torch.exp(d.double())[:, None] * dot(1, 0) * v[:, :, 0]], 2)
    rows = [x.double() for x in (q, k, v)]
    within(out, formula(*rows), formula(*(x.abs() for x in rows)), 2 * E + 192, "out")


def test_one_step_of_many_heads_with_gradients(fwp):
    N, E = 1 << 15, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(N, 1, 1, E, generator=g, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    go = torch.randn(N, 1, 1, E, generator=g, device="cuda").bfloat16()
    grads = torch.autograd.grad(fwp.decayed_sum(q, k, v, torch.full((1,), -0.5, device="cuda")), (q, k, v), go)
    q, k, v, go = (x.detach().double() for x in (q, k, v, go))
    dot = lambda a, b: (a * b).sum(-1, keepdim=True)
    for got, name, (x, a, b) in zip(grads, "qkv", ((k, go, v), (q, go, v), (go, q, k))):
        within(got, x * dot(a, b), x.abs() * dot(a.abs(), b.abs()), 8 * E + 512, name)
