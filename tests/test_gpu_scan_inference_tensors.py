"""A call that cannot be recorded, since autograd keeps no tensor of inference mode, is refused before its state goes on; one whose tensors are copied for their layout,
or that records nothing, is an ordinary call."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tensors():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    return dict(X=r(2, 3, 9, 8), weight=r(3, 8, 4), bias=r(3, 8)), dict(Q=r(2, 3, 9, 16), K=r(2, 3, 9, 16), V=r(2, 3, 9, 8), delta=r(2, 3, 9, 8), A=-r(3, 16, 8).abs(),
                                                                         D=r(3, 8), Z=r(2, 3, 9, 8), delta_bias=r(3, 8)), r(2, 3, 3, 8), r(2, 3, 16, 8)


@pytest.mark.parametrize("op,name", [("causal_conv", k) for k in ("X", "bias", "lengths")] + [("selective_scan", k) for k in ("Q", "V", "A", "D", "Z", "lengths")])
def test_refused_with_the_state_as_it_was(fwp, op, name):
    conv, scan, conv_state, W = tensors()
    call, state, kept, leaf = (conv, "state", conv_state, "weight") if op == "causal_conv" else (scan, "W", W, "K")
    call["lengths"] = torch.tensor([9, 4]).cuda()
    f = getattr(fwp, op)
    with torch.inference_mode():
        call[name] = call[name].clone()
    call[leaf] = call[leaf].requires_grad_()
    before = kept.clone()
    with pytest.raises(fwp._lib.FwpError, match="inference"):
        f(**call, **{state: kept}, softplus=True) if op == "selective_scan" else f(**call, **{state: kept})
    assert torch.equal(kept, before)
    with torch.no_grad():
        f(**call, **{state: kept})
    assert not torch.equal(kept, before)


def test_copies_are_ordinary(fwp):
    conv, _, state, _ = tensors()
    want = fwp.causal_conv(**conv, state=state.clone())
    with torch.inference_mode():
        x = conv["X"].transpose(2, 3).contiguous().transpose(2, 3)      # the last axis apart: read from a copy
    w = conv["weight"].clone().requires_grad_()
    out = fwp.causal_conv(x, w, conv["bias"], state)
    assert torch.equal(out, want) and torch.autograd.grad(out.sum(), w)[0].abs().sum() > 0
