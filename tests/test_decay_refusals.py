"""What the operators of the decayed sum rule's block refuse, on the CPU: shapes, types and strides are compared before the device is looked at, and the C entry points
check their arguments before anything is launched.  And the formulas that their GPU tests go by, against differences."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as ad

import decay_formulas as F


def rows(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


LENGTHS = torch.zeros(2, dtype=torch.int64)


def sum_call(fwp, **change):
    t = dict(Q=rows(2, 2, 5, 16), K=rows(2, 4, 5, 16), V=rows(2, 4, 5, 8), log_decay=rows(2, 4, 5), W=rows(2, 4, 16, 8), lengths=LENGTHS)
    t.update(change)
    return fwp.decayed_sum(**t)


def rotary_call(fwp, **change):
    t = dict(Q=rows(2, 4, 5, 16), K=rows(2, 1, 5, 16), frequencies=rows(8, dtype=torch.float64), positions=LENGTHS, lengths=LENGTHS)
    t.update(change)
    return fwp.rotary(**t)


def norm_call(fwp, **change):
    t = dict(X=rows(4, 6, 24), groups=3, weight=rows(24), bias=rows(24), gate=rows(4, 6, 24), activation="silu")
    t.update(change)
    return fwp.group_norm(**t)


SUM = [(dict(Q=rows(2, 5, 16)), "4-D"), (dict(V=rows(2, 5, 8)), "4-D"), (dict(log_decay=rows(2, 4)), "log_decay"), (dict(log_decay=rows(2, 4, 6)), "log_decay"),
       (dict(log_decay=rows(4, 5, 2).permute(2, 0, 1).double()), "must be fp32"), (dict(log_decay=rows(3)), "must divide"), (dict(log_decay=rows(2, 3, 5)), "must divide"),
       (dict(Q=rows(2, 3, 5, 16)), "heads of Q"), (dict(K=rows(2, 4, 5, 15)), "K"), (dict(K=rows(1, 4, 5, 16)), "K"), (dict(V=rows(2, 4, 4, 8)), "V"),
       (dict(K=rows(2, 4, 5, 16, dtype=torch.float16)), "K must have the type"), (dict(V=rows(2, 4, 5, 8, dtype=torch.bfloat16)), "V must have the type"),
       (dict(Q=rows(2, 2, 5, 16, dtype=torch.float64)), "fp32, fp16 or bf16"), (dict(Q=rows(2, 2, 5, 129), K=rows(2, 4, 5, 129)), "at most 128"),
       (dict(V=rows(2, 4, 5, 65537)), "65536"), (dict(W=rows(2, 4, 8, 16)), "W must be"), (dict(W=rows(2, 4, 16, 8, dtype=torch.bfloat16)), "W must be"),
       (dict(W=rows(2, 4, 8, 16).transpose(2, 3)), "W must be"), (dict(lengths=torch.zeros(2)), "lengths"), (dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths"),
       (dict(Q=rows(2, 2, 0, 16), K=rows(2, 4, 0, 16), V=rows(2, 4, 0, 8), log_decay=rows(4)), "at least 1"), (dict(Q=rows(2, 0, 5, 16)), "at least 1"),
       (dict(log_decay=rows(0)), "at least 1"), (dict(), "MI355X")]
ROTARY = [(dict(Q=rows(4, 5, 16)), "4-D"), (dict(K=rows(4, 5, 16)), "4-D"), (dict(K=rows(2, 1, 5, 8)), "K"), (dict(K=rows(2, 1, 4, 16)), "K"),
          (dict(K=rows(2, 1, 5, 16, dtype=torch.float16)), "K must have"), (dict(Q=rows(2, 4, 5, 16, dtype=torch.int32)), "fp32, fp16 or bf16"),
          (dict(frequencies=rows(8)), "fp64"), (dict(frequencies=rows(8, 1, dtype=torch.float64)), "fp64"), (dict(frequencies=rows(9, dtype=torch.float64)), "1 to D / 2"),
          (dict(frequencies=rows(0, dtype=torch.float64)), "1 to D / 2"), (dict(frequencies=rows(8, dtype=torch.float64).requires_grad_()), "no gradient of the frequencies"),
          (dict(positions=torch.zeros(2, dtype=torch.int32)), "positions"), (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
          (dict(positions=torch.zeros(2, 4, dtype=torch.int64)), "positions"), (dict(lengths=torch.zeros(2)), "lengths"),
          (dict(Q=rows(2, 4, 0, 16), K=None), "at least 1"), (dict(K=rows(2, 0, 5, 16)), "at least 1"), (dict(), "MI355X"), (dict(K=None, positions=None), "MI355X")]
NORM = [(dict(X=torch.zeros(())), "channels"), (dict(groups=5), "multiple of the groups"), (dict(groups=0), "multiple of the groups"), (dict(groups=-3), "multiple of the groups"),
        (dict(X=rows(4, 6, 24, dtype=torch.float64)), "fp32, fp16 or bf16"), (dict(gate=rows(4, 6, 23)), "gate"), (dict(gate=rows(4, 1, 24)), "gate"),
        (dict(gate=rows(4, 6, 24, dtype=torch.float16)), "gate must have"), (dict(weight=rows(8)), "weight"), (dict(bias=rows(1, 24)), "bias"),
        (dict(weight=rows(24, dtype=torch.bfloat16)), "weight must be fp32"), (dict(activation="relu"), "activation"),
        (dict(X=rows(2, 1025), groups=1, weight=None, bias=None, gate=None), "1024"), (dict(X=rows(1, 65600), groups=656, weight=None, bias=None, gate=None), "65536"),
        (dict(X=rows(0, 24), gate=None), "at least 1"), (dict(X=rows(3, 0), gate=None), "at least 1"), (dict(), "MI355X")]


@pytest.mark.parametrize("call,change,message", [(f, *c) for f, cases in ((sum_call, SUM), (rotary_call, ROTARY), (norm_call, NORM)) for c in cases])
def test_refusals(fwp, call, change, message):
    with pytest.raises(fwp._lib.FwpError, match=message):
        call(fwp, **change)


@pytest.mark.parametrize("call,name", [(sum_call, "Q"), (sum_call, "log_decay"), (sum_call, "W"), (rotary_call, "K"), (rotary_call, "frequencies"), (norm_call, "X"),
                                       (norm_call, "gate"), (norm_call, "weight")])
def test_tensors_with_a_tangent_are_refused(fwp, call, name):
    shapes = dict(Q=(2, 2, 5, 16), log_decay=(2, 4, 5), W=(2, 4, 16, 8), K=(2, 1, 5, 16), frequencies=(8,), X=(4, 6, 24), gate=(4, 6, 24), weight=(24,))
    t = rows(*shapes[name], dtype=torch.float64 if name == "frequencies" else torch.float32)
    with ad.dual_level():
        with pytest.raises(fwp._lib.FwpError, match="tangent"):
            call(fwp, **{name: ad.make_dual(t, torch.ones_like(t))})


def test_frequencies_refuse(fwp):
    for args in (dict(width=7), dict(width=0), dict(width=8, scaling="none"), dict(width=8, scaling="parts"), dict(width=8, factor=0.0), dict(width=8, base=-1.0),
                 dict(width=8, scaling="parts", trained=100, turns=(2.0, 2.0))):
        with pytest.raises(fwp._lib.FwpError):
            fwp.rotary_frequencies(**args)


def test_an_operator_without_its_binding_says_so(fwp, monkeypatch):
    import importlib
    monkeypatch.setattr(importlib.import_module(fwp.__name__ + ".selective_scan"), "_fwp_torch", None)
    for call in (sum_call, rotary_call, norm_call):
        with pytest.raises(fwp._lib.FwpError, match="build_torch.sh"):
            call(fwp)


def test_layers_refuse(fwp):
    with pytest.raises(ValueError, match="even"):
        fwp.DecayedSumLayer(2, 16, 7)
    with pytest.raises(ValueError, match="own operator"):
        fwp.DecayedSumDecoderLayer(2, 16, 8, 32, fast_weight_op=fwp.fast_weight_delta)
    with pytest.raises(ValueError, match="carry_over"):
        fwp.DecayedSumLayer(2, 16, 8)(torch.zeros(3, 2, 16), mems=(None, None))


def test_c_entry_points_refuse_before_any_launch(fwp):
    L = fwp._lib
    lib = L.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    v, out, none, no_out = L.View(4096, 640, 80, 16), L.OutView(4096, 640, 80, 16), L.View(0, 0, 0, 0), L.OutView(0, 0, 0, 0)
    far = L.View(4096, 640, 80, (1 << 24) + 1)
    E_NULL, E_SHAPE = -1, -2
    args = lambda **k: ctypes.byref(L.DecayedSumArgs(**{**dict(q=v, k=v, v=v, decay=4096, dN=40, dH=5, dL=1, scale=1.0, N=2, H=8, L=5, E=16, M=16, HQ=8, HK=8, HV=8), **k}))
    assert lib.fwp_decayed_sum_fwd(None, p, out, None, None, None) == E_NULL
    for bad in (dict(q=none), dict(k=none), dict(v=none), dict(decay=0), dict(decay=4098), dict(q=L.View(4098, 1, 1, 1))):
        assert lib.fwp_decayed_sum_fwd(args(**bad), p, out, None, None, None) == E_NULL, bad
    for bad in (dict(type=3), dict(N=0), dict(H=0), dict(L=0), dict(E=0), dict(M=0), dict(E=129), dict(M=65537), dict(HQ=3), dict(HK=0), dict(HV=16), dict(per_head=1),
                dict(N=1 << 20, H=1 << 12, HQ=1, HK=1, HV=1), dict(k=far), dict(L=(1 << 30) + 1)):
        assert lib.fwp_decayed_sum_fwd(args(**bad), p, out, None, None, None) == E_SHAPE, bad
        assert lib.fwp_decayed_sum_workspace(args(**bad), 0) == E_SHAPE, bad
    assert lib.fwp_decayed_sum_fwd(args(), p, no_out, None, None, None) == E_NULL
    assert lib.fwp_decayed_sum_fwd(args(), p, out, odd, None, None) == E_NULL
    assert lib.fwp_decayed_sum_fwd(args(), p, L.OutView(4096, 640, 80, 1 << 25), None, None, None) == E_SHAPE
    # a sequence cut into segments needs its workspace
    assert lib.fwp_decayed_sum_workspace(args(N=1, H=1, L=100000, HQ=1, HK=1, HV=1), 0) > 0
    assert lib.fwp_decayed_sum_fwd(args(N=1, H=1, L=100000, HQ=1, HK=1, HV=1), p, out, None, None, None) == E_NULL
    bwd = lambda a=None, saved=p, go=v, gq=out, gd=p, work=p: lib.fwp_decayed_sum_bwd(a or args(), saved, go, gq, out, out, gd, work, None)
    for bad in (dict(saved=None), dict(saved=odd), dict(go=none), dict(gq=no_out), dict(gd=None), dict(work=odd)):
        assert bwd(**bad) == E_NULL, bad
    assert bwd(a=args(HQ=4), work=None) == E_NULL and bwd(go=far) == E_SHAPE and bwd(a=args(E=0)) == E_SHAPE
    assert lib.fwp_decayed_sum_saved_floats(0, 1, 1, 64, 16, 16) == 2 * 32 * 32 and lib.fwp_decayed_sum_saved_floats(0, 1, 1, 64, 129, 16) == E_SHAPE

    turn = lambda **k: ctypes.byref(L.RotaryArgs(**{**dict(q=v, k=v, frequencies=4096, scale=1.0, N=2, HQ=8, HK=8, L=5, D=16, pairs=8), **k}))
    assert lib.fwp_rotary(None, out, out, None) == E_NULL
    for bad in (dict(q=none), dict(frequencies=0), dict(frequencies=4100)):
        assert lib.fwp_rotary(turn(**bad), out, out, None) == E_NULL, bad
    for bad in (dict(type=-1), dict(N=0), dict(HQ=0), dict(HK=0), dict(L=0), dict(D=0), dict(pairs=0), dict(pairs=9), dict(D=65537)):
        assert lib.fwp_rotary(turn(**bad), out, out, None) == E_SHAPE, bad
    assert lib.fwp_rotary(turn(), no_out, out, None) == E_NULL and lib.fwp_rotary(turn(), out, no_out, None) == E_NULL

    norm = lambda **k: ctypes.byref(L.GroupNormArgs(**{**dict(x=4096, gate=4096, x_step=64, gate_step=64, weight=4096, bias=4096, eps=1e-5, act=2, rows=4, groups=4, size=16), **k}))
    assert lib.fwp_group_norm_fwd(None, p, None) == E_NULL and lib.fwp_group_norm_fwd(norm(x=0), p, None) == E_NULL and lib.fwp_group_norm_fwd(norm(), None, None) == E_NULL
    for bad in (dict(type=3), dict(act=3), dict(rows=0), dict(groups=0), dict(size=0), dict(size=1025), dict(groups=5000)):
        assert lib.fwp_group_norm_fwd(norm(**bad), p, None) == E_SHAPE, bad
        assert lib.fwp_group_norm_bwd(norm(**bad), p, p, p, p, p, p, None) == E_SHAPE, bad
    for bad in ((None, p, p, p, p, p), (p, None, p, p, p, p), (p, p, None, p, p, p), (p, p, p, p, p, None), (p, p, p, None, p, None)):
        assert lib.fwp_group_norm_bwd(norm(), *bad, None) == E_NULL, bad
    assert lib.fwp_group_norm_bwd(norm(gate=0), p, p, p, p, p, p, None) == E_NULL
    assert lib.fwp_group_norm_workspace(0, 4, 4, 16) >= 2 * 64 and lib.fwp_group_norm_workspace(0, 0, 4, 16) == E_SHAPE


def test_more_rows_than_a_walk_counts_are_refused(fwp):
    """Rows go on in steps of up to 4096: the last ones below 2^31 have no next one in 32 bits"""
    L = fwp._lib
    lib, p = L.lib(), ctypes.c_void_p(4096)
    norm = lambda rows: ctypes.byref(L.GroupNormArgs(x=4096, x_step=1, weight=4096, bias=4096, eps=1e-5, rows=rows, groups=1, size=1))
    for rows in ((1 << 30) + 1, (1 << 31) - 1):
        assert lib.fwp_group_norm_fwd(norm(rows), p, None) == -2
        assert lib.fwp_group_norm_bwd(norm(rows), p, p, None, p, p, p, None) == -2
        assert lib.fwp_group_norm_workspace(0, rows, 1, 1) == -2
    assert lib.fwp_group_norm_workspace(0, 1 << 30, 1, 1) > 0


def test_plans_of_long_sequences_are_quick(fwp):
    """A call asks for its plan several times: those of one sequence of a million steps, which may have thousands of segments, within a millisecond each"""
    import time
    L = fwp._lib
    lib = L.lib()
    v = L.View(4096, 1 << 30, 1 << 30, 16)
    a = ctypes.byref(L.DecayedSumArgs(q=v, k=v, v=v, decay=4096, dN=1 << 20, dH=1 << 20, dL=1, scale=1.0, N=1, H=1, L=1 << 20, E=16, M=16, HQ=1, HK=1, HV=1))
    for backward in (0, 1):
        assert lib.fwp_decayed_sum_workspace(a, backward) > 0
        start = time.perf_counter()
        for _ in range(100):
            lib.fwp_decayed_sum_workspace(a, backward)
        assert time.perf_counter() - start < 0.1


@pytest.mark.parametrize("per_head", [True, False])
def test_the_formulas_gradients_against_differences(per_head):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    t = dict(q=rnd(2, 1, 9, 5), k=rnd(2, 2, 9, 5), v=rnd(2, 4, 9, 3), g=-rnd(*((4,) if per_head else (2, 4, 9))).abs())
    go, n, W = rnd(2, 4, 9, 3), torch.tensor([9, 6]), rnd(2, 4, 5, 3)
    value = lambda a: (F.decayed_sum(**a, W=W, scale=0.7, lengths=n)[0] * go).sum()
    grads = F.decayed_sum(**t, W=W, scale=0.7, lengths=n, go=go)[2:]
    for name, grad in zip(t, grads):
        v = rnd(*t[name].shape)
        slope = (value({**t, name: t[name] + 1e-6 * v}) - value({**t, name: t[name] - 1e-6 * v})) / 2e-6
        assert abs(float(slope - (grad * v).sum())) <= 1e-6 * (1 + abs(float(slope))), name
