"""A decayed sum layer that is built without memory (device "meta"), given some and then filled, as large models are."""
import pytest
import torch

import decay_formulas as F


def build(fwp, device):
    with torch.device(device):
        return fwp.DecayedSumLayer(3, 48, 16, token_decay=True)


def test_frequencies_are_numbers_wherever_a_layer_is_built(fwp):
    for device in ("cpu", "meta"):
        f = build(fwp, device)._frequencies
        # made by another power than the formula's: two roundings of 64 bits each
        assert f.device.type == "cpu" and f.dtype is torch.float64 and torch.allclose(f, F.frequencies(16), rtol=1e-15, atol=0.0)
    layer = build(fwp, "meta").to_empty(device="cpu")
    layer.reset_decay_parameters()
    assert torch.equal(layer.decay_logit, build(fwp, "cpu").decay_logit)


@pytest.mark.gpu
def test_a_layer_that_is_filled_later(fwp):
    torch.manual_seed(0)
    want = build(fwp, "cpu").cuda()
    got = build(fwp, "meta").to_empty(device="cuda")
    got.load_state_dict(want.state_dict())
    h = torch.randn(20, 2, 48).cuda()
    with torch.no_grad():
        assert torch.equal(got(h), want(h))
