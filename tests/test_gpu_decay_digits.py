"""The decayed sum rule in fp32: how many roundings a long sequence's state passes.

A rounding is off by 2^-24 / sqrt(3) of the number in the root mean square at most, and roundings of different steps add up as a random walk.  Of 1024 steps in 32 chunks, the state is
rounded once a chunk (32); a chunk's own sum, the sum over 32 keys or columns, that over the steps of a chunk and the scores' come four terms at a time (8 each).  That is 64 of them (some more where 64 keys go
in six products of parts, 32 terms at a time): 8 x 2^-24 / sqrt(3) = 2.75e-7 of a result's norm.  Were every product of a chunk added to the state by itself, it would be 8 x 32 for the state alone."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_decay_carried import formulas

MOST = 8 * 2.0 ** -24 / 3 ** 0.5


@pytest.mark.parametrize("E,M", [(32, 32), (32, 64), (64, 64)])
def test_a_chunk_rounds_the_state_once(fwp, E, M):
    N, H, L = 8, 8, 1024
    g = torch.Generator(device="cuda").manual_seed(E + M)
    q, k, v, go = (torch.randn(N, H, L, d, generator=g, device="cuda") for d in (E, E, M, M))
    decay = torch.log1p(-torch.exp2(-5.0 - torch.arange(H, device="cuda")))      # memories of 32 to 4096 steps
    leaves = [x.double().requires_grad_() for x in (q, k, v)]
    out, _ = formulas(*leaves, decay.double()[None, :, None].expand(N, H, L), torch.zeros(N, H, E, M, device="cuda", dtype=torch.float64), E ** -0.5)
    want = [out.detach(), *torch.autograd.grad(out, leaves, go.double())]
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = fwp.decayed_sum(*leaves, decay, scale=E ** -0.5)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    for name, a, b in zip(("out", "Q", "K", "V"), got, want):
        assert float((a.double() - b).norm()) <= MOST * float(b.norm()), name
