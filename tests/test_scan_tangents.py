"""Forward-mode differentiation of the selective state space block's operators is refused, whichever tensor has the tangent: it would be lost
otherwise.  On the CPU, since arguments are looked at before the device is."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

r = torch.zeros
CALLS = {
    "causal_conv": dict(X=r(2, 3, 5, 8), weight=r(3, 8, 4), bias=r(3, 8), state=r(2, 3, 3, 8)),
    "selective_scan": dict(Q=r(2, 3, 5, 16), K=r(2, 3, 5, 16), V=r(2, 3, 5, 8), delta=r(2, 3, 5, 8), A=r(3, 16, 8), W=r(2, 3, 16, 8), D=r(3, 8), Z=r(2, 3, 5, 8),
                           delta_bias=r(3, 8)),
    "residual_norm": dict(y=r(4, 6, 8), x=r(4, 6, 8), after=r(8), gate=r(4, 6, 8), scale=r(8), before=r(8)),
}


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("op,name", [(op, name) for op, call in CALLS.items() for name in call])
def test_a_tangent_is_refused(fwp, op, name, grads):
    call = dict(CALLS[op])
    if grads:       # another tensor of the call is recorded for a backward pass
        other = next(k for k in call if k != name)
        call[other] = call[other].clone().requires_grad_()
    with fwAD.dual_level():
        call[name] = fwAD.make_dual(call[name], torch.ones_like(call[name]))
        with pytest.raises(fwp._lib.FwpError, match="forward-mode"):
            getattr(fwp, op)(**call)


@pytest.mark.parametrize("op", CALLS)
def test_ordinary_tensors_inside_a_level_are_ordinary(fwp, op):
    with fwAD.dual_level(), pytest.raises(fwp._lib.FwpError, match="MI355X"):      # the next check
        getattr(fwp, op)(**CALLS[op])


def test_a_function_transform_is_refused(fwp):
    f = lambda x: fwp.causal_conv(x, CALLS["causal_conv"]["weight"])
    with pytest.raises(fwp._lib.FwpError, match="forward-mode"):
        torch.func.jvp(f, (r(2, 3, 5, 8),), (torch.ones(2, 3, 5, 8),))
