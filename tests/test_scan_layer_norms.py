"""The norms of SelectiveScanDecoderLayer are modules like any other: replaced, hooked to, without weights or with an epsilon of its own, each is what
is computed.  On the CPU with the formula in the operator's place, in 64 bits; on the GPU with the operator.

Tolerance on the GPU: the two residual norms, the two products and the norm in front are fewer than 1024 roundings of 2^-24 one after the other, each of
terms that are up to 64 times the largest result (a norm's rows have terms of up to sqrt(cols) = 7, and two norms follow one another)."""
import copy
import importlib

import pytest
import torch
from torch import nn

import scan_formulas as F

COLS = 48


class Mixer(nn.Module):
    """In the scan's place: takes the call of a SelectiveScanLayer"""

    def __init__(self):
        super().__init__()
        self.net = nn.Linear(COLS, COLS)

    def forward(self, h, attn_mask=None, mems=None, carry_over_fast_weight=False, lengths=None):
        return self.net(h)


class Rms(nn.Module):
    def __init__(self):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(COLS))

    def forward(self, x):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * self.weight


def formula(y, x, after=None, gate=None, scale=None, before=None, eps=1e-5, rms=False, activation=None):
    pair = lambda n: n if isinstance(n, tuple) else (n, None)
    return F.residual_norm(y, x, *pair(after), gate, scale, *pair(before), eps, rms, activation)


def layer_of(fwp):
    torch.manual_seed(3)
    m = fwp.SelectiveScanDecoderLayer(4, COLS, COLS // 4, 2 * COLS)
    m.dec_attn = Mixer()
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p))
    return m


def by_modules(m, h):
    a = m.dec_attn(m.norm_in(h))
    r = h + m.scale_attn * m.norm_attn(a)
    return r + m.scale_ff * m.norm_ff(m.ff(m.norm_mid(r)))


def replaced(name, make):
    return lambda m: setattr(m, name, make())


def hooked(name):
    return lambda m: getattr(m, name).register_forward_hook(lambda mod, args, out: 2 * out)


def epsilon(name, eps):
    return lambda m: setattr(getattr(m, name), "eps", eps)


def changed_forward(m):
    forward = m.norm_ff.forward
    m.norm_ff.forward = lambda x: forward(x) - 1


NORMS = ["norm_in", "norm_attn", "norm_mid", "norm_ff"]
CHANGES = {"as it is": lambda m: None, "forward": changed_forward}
for norm in NORMS:
    CHANGES |= {f"{norm} identity": replaced(norm, nn.Identity), f"{norm} rms": replaced(norm, Rms), f"{norm} hook": hooked(norm), f"{norm} eps": epsilon(norm, 0.3),
                f"{norm} bare": replaced(norm, lambda: nn.LayerNorm(COLS, elementwise_affine=False)),
                f"{norm} no bias": replaced(norm, lambda: nn.LayerNorm(COLS, bias=False)),
                f"{norm} halves": replaced(norm, lambda: nn.Sequential(nn.Unflatten(-1, (2, COLS // 2)), nn.LayerNorm(COLS // 2), nn.Flatten(-2)))}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def compare(fwp, monkeypatch, m, device, change=lambda m: None):
    h = torch.randn(7, 3, COLS, dtype=torch.float64)
    ref = copy.deepcopy(m)
    change(m), change(ref)
    ref.double()
    want = by_modules(ref, h)
    if device == "cpu":
        monkeypatch.setattr(importlib.import_module(fwp.__name__ + ".layers"), "residual_norm", formula)
        assert torch.allclose(m.double()(h), want, rtol=1e-10, atol=1e-10)
    else:
        got = m.cuda()(h.float().cuda())
        exact = by_modules(ref, h.float().double())
        assert float((got.cpu().double() - exact).abs().max()) <= 1024 * 64 * F.EPS32 * float(exact.abs().max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", CHANGES)
def test_each_norm_is_the_module_that_is_there(fwp, monkeypatch, change, device):
    compare(fwp, monkeypatch, layer_of(fwp), device, CHANGES[change])


@pytest.mark.parametrize("device", DEVICES)
def test_global_hooks_see_every_norm(fwp, monkeypatch, device):
    m, seen = layer_of(fwp), []
    handle = nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(mod))
    try:
        compare(fwp, monkeypatch, m, device)
    finally:
        handle.remove()
    assert all(any(x is getattr(m, n) for x in seen) for n in NORMS)


@pytest.mark.parametrize("device", DEVICES)
def test_an_untouched_layer_takes_two_operators(fwp, monkeypatch, device):
    m, calls = layer_of(fwp).to(device), []
    layers = importlib.import_module(fwp.__name__ + ".layers")
    real = formula if device == "cpu" else layers.residual_norm
    monkeypatch.setattr(layers, "residual_norm", lambda *a, **k: (calls.append(k), real(*a, **k))[1])
    m(torch.randn(5, 2, COLS, device=device))
    assert [("after" in k, "before" in k) for k in calls] == [(True, True), (True, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("change", ["norm_attn hook", "norm_mid eps", "norm_ff rms", "norm_mid identity"])
def test_under_autocast(fwp, change, dtype):
    """About sixteen roundings of the narrow type lie on the way: the products' operands and results, and those of the residual norms beside them."""
    m = layer_of(fwp)
    ref = copy.deepcopy(m)
    CHANGES[change](m), CHANGES[change](ref)
    h = torch.randn(7, 3, COLS)
    want = by_modules(ref.double(), h.double())
    m = m.cuda()
    with torch.autocast("cuda", dtype):
        got = m(h.cuda())
    got.square().mean().backward()
    assert got.dtype is torch.float32 and float((got.cpu().double() - want).norm()) <= 16 * F.half_step(dtype) * float(want.norm())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
