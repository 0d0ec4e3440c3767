"""Views whose sign is still to be changed (the imaginary part of a conjugate): the selective state space block's operators take their values, not what
their memory holds, and refuse one as a state that they would write to."""
import pytest
import torch

SHAPE = (2, 3, 20, 1)


def negated(t):
    """The same values in memory of the other sign, as contiguous as t"""
    return torch._neg_view(-t)


def imaginary(t):
    return torch.complex(torch.zeros_like(t), -t).conj().imag


def test_states_are_refused(fwp):
    r = torch.zeros
    for state in (negated(r(2, 3, 3, 1)), imaginary(r(1, 1, 1, 1))):
        n, h, k, d = state.shape
        with pytest.raises(fwp._lib.FwpError, match="state must be contiguous"):
            fwp.causal_conv(r(n, h, 20, d), r(h, d, k + 1), state=state)
    with pytest.raises(fwp._lib.FwpError, match="W must be"):
        fwp.selective_scan(r(SHAPE), r(SHAPE), r(SHAPE), r(SHAPE), r(3, 1, 1), negated(r(2, 3, 1, 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("view", [negated, imaginary])
def test_values_are_those_of_the_view(fwp, view):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    calls = {
        fwp.causal_conv: [r(SHAPE), r(3, 1, 4), r(3, 1)],
        lambda q, k, v, delta, A, D, z, bias: fwp.selective_scan(q, k, v, delta, A, D=D, Z=z, delta_bias=bias, softplus=True):
            [r(SHAPE), r(SHAPE), r(SHAPE), r(SHAPE), -r(3, 1, 1).abs(), r(3, 1), r(SHAPE), r(3, 1)],
        lambda y, x, gate, after, scale, before: sum(fwp.residual_norm(y, x, after=after, gate=gate, scale=scale, before=before, activation="silu")):
            [r(7, 40), r(7, 40), r(7, 1), r(40), r(40), r(40)],
    }
    for f, args in calls.items():
        want = f(*args)
        for i in range(len(args)):
            seen = view(args[i])
            assert seen.is_neg() and torch.equal(seen, args[i])
            assert torch.equal(f(*args[:i], seen, *args[i + 1:]), want), i
        leaf = args[0].clone().requires_grad_()
        go = torch.randn(want.shape, generator=g).cuda()
        out = f(leaf, *args[1:])
        a, = torch.autograd.grad(out, leaf, go, retain_graph=True)
        b, = torch.autograd.grad(out, leaf, view(go))
        assert torch.equal(a, b)
