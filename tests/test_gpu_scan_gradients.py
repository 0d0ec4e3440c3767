"""Gradients of the selective state space block's parameters have memory of their own: one that is saved, resized or freed takes no other with it."""
import io

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def calls(fwp):
    r = lambda *s: torch.randn(*s).cuda()
    p = lambda *s: (torch.randn(*s) / 4).cuda().requires_grad_()
    w, b = p(2, 24, 4), p(2, 24)
    yield [w, b], fwp.causal_conv(r(3, 2, 20, 24), w, b, silu=True)
    A, D, bias = (-torch.rand(2, 8, 24)).cuda().requires_grad_(), p(2, 24), p(2, 24)
    yield [A, D, bias], fwp.selective_scan(r(3, 2, 20, 8), r(3, 2, 20, 8), r(3, 2, 20, 24), r(3, 2, 20, 24), A, D=D, delta_bias=bias, softplus=True)
    five = [p(131) for _ in range(5)]
    y, n = fwp.residual_norm(r(9, 131), r(9, 131), after=tuple(five[:2]), scale=five[2], before=tuple(five[3:]))
    yield five, y + n


def test_no_two_gradients_share_memory(fwp):
    torch.manual_seed(0)
    for params, out in calls(fwp):
        out.square().sum().backward()
        stores = [x.grad.untyped_storage() for x in params]
        assert len({s.data_ptr() for s in stores}) == len(params)
        for x, s in zip(params, stores):
            assert x.grad.is_contiguous() and s.nbytes() == 4 * x.numel()
            buffer = io.BytesIO()
            torch.save(x.grad, buffer)
            assert len(buffer.getvalue()) < 4 * x.numel() + 2048
