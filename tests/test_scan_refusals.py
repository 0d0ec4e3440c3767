"""What the operators of the selective state space block refuse, on the CPU: shapes, types and strides are compared before the device is looked at, and the C
entry points check their arguments before anything is launched.  And the formulas that their GPU tests go by, against differences."""
import ctypes

import pytest
import torch

import scan_formulas as F


def rows(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def conv_call(fwp, **change):
    t = dict(X=rows(2, 3, 5, 8), weight=rows(3, 8, 4), bias=rows(3, 8), state=rows(2, 3, 3, 8), lengths=torch.zeros(2, dtype=torch.int64))
    t.update(change)
    return fwp.causal_conv(**t)


def scan_call(fwp, **change):
    t = dict(Q=rows(2, 3, 5, 16), K=rows(2, 3, 5, 16), V=rows(2, 3, 5, 8), delta=rows(2, 3, 5, 8), A=rows(3, 16, 8), W=rows(2, 3, 16, 8), D=rows(3, 8),
             Z=rows(2, 3, 5, 8), delta_bias=rows(3, 8), lengths=torch.zeros(2, dtype=torch.int64))
    t.update(change)
    return fwp.selective_scan(**t)


def norm_call(fwp, **change):
    t = dict(y=rows(4, 6, 8), x=rows(4, 6, 8), after=(rows(8), rows(8)), gate=rows(4, 6, 8), scale=rows(8), before=(rows(8), rows(8)), activation="silu")
    t.update(change)
    return fwp.residual_norm(**t)


CONV = [(dict(X=rows(2, 5, 8)), "4-D"), (dict(X=rows(2, 3, 0, 8)), "at least 1"), (dict(X=rows(2, 3, 5, 8, dtype=torch.float64)), "fp32, fp16 or bf16"),
        (dict(weight=rows(8, 4)), "weight"), (dict(weight=rows(3, 8, 9)), "1 to 8 taps"), (dict(weight=rows(3, 7, 4)), "weight"),
        (dict(weight=rows(3, 8, 0)), "taps"), (dict(weight=rows(3, 8, 4, dtype=torch.float16)), "weight must be fp32"), (dict(bias=rows(8)), "bias"),
        (dict(state=rows(2, 3, 4, 8)), "state"), (dict(state=rows(2, 3, 3, 8, dtype=torch.bfloat16)), "state"),
        (dict(state=rows(2, 3, 8, 3).transpose(2, 3)), "contiguous"), (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths"),
        (dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths"), (dict(), "MI355X")]
SCAN = [(dict(Q=rows(2, 3, 16)), "4-D"), (dict(K=rows(2, 3, 5, 8)), "K"), (dict(K=rows(2, 3, 4, 16)), "K"), (dict(V=rows(2, 3, 4, 8)), "V"),
        (dict(delta=rows(2, 3, 5, 1)), "delta"), (dict(Z=rows(2, 3, 5, 9)), "Z"), (dict(Z=rows(2, 3, 5, 8, dtype=torch.float16)), "Z must have the type"),
        (dict(Q=rows(2, 3, 5, 65), K=rows(2, 3, 5, 65)), "at most 64"), (dict(A=rows(3, 8, 16)), "A"), (dict(A=rows(16, 8)), "A"), (dict(D=rows(8)), "D"),
        (dict(delta_bias=rows(3, 9)), "delta_bias"), (dict(W=rows(2, 3, 8, 16)), "W must be"), (dict(W=rows(2, 3, 16, 8, dtype=torch.bfloat16)), "W must be"),
        (dict(W=rows(2, 3, 8, 16).transpose(2, 3)), "W must be"), (dict(lengths=torch.zeros(2)), "lengths"),
        (dict(**{k: rows(2, 3, 0, n) for k, n in (("Q", 16), ("K", 16), ("V", 8), ("delta", 8), ("Z", 8))}), "at least 1"), (dict(), "MI355X")]
NORM = [(dict(x=rows(4, 6, 9)), "x"), (dict(x=rows(4, 6, 8, dtype=torch.float16)), "x must be fp32"), (dict(y=rows(4, 6, 8, dtype=torch.int32)), "y must be"),
        (dict(gate=rows(4, 6, 2)), "gate"), (dict(gate=rows(4, 1, 8)), "gate"), (dict(gate=rows(4, 6, 8, dtype=torch.bfloat16)), "gate must have the type"),
        (dict(scale=rows(1)), "scale"), (dict(after=rows(7)), "after"), (dict(after=(None, rows(8))), "without its weight"),
        (dict(before=(rows(8), rows(9))), "before"), (dict(before=(rows(8), rows(8), rows(8))), "pair"), (dict(activation="relu"), "activation"),
        (dict(y=rows(2, 8193), x=rows(2, 8193), after=None, gate=None, scale=None, before=None), "8192"),
        (dict(y=rows(0, 8), x=rows(0, 8), gate=None), "at least 1"), (dict(), "MI355X")]


@pytest.mark.parametrize("call,change,message", [(f, *c) for f, cases in ((conv_call, CONV), (scan_call, SCAN), (norm_call, NORM)) for c in cases])
def test_refusals(fwp, call, change, message):
    with pytest.raises(fwp._lib.FwpError, match=message):
        call(fwp, **change)


def test_an_operator_without_its_binding_says_so(fwp, monkeypatch):
    import importlib
    module = importlib.import_module(fwp.__name__ + ".selective_scan")
    monkeypatch.setattr(module, "_fwp_torch", None)
    with pytest.raises(fwp._lib.FwpError, match="build_torch.sh"):
        conv_call(fwp)


def test_c_entry_points_refuse_before_any_launch(fwp):
    L = fwp._lib
    lib = L.lib()
    p, null = ctypes.c_void_p(4096), L.View(0, 0, 0, 0)
    v, out, none = L.View(4096, 64, 32, 8), L.OutView(4096, 64, 32, 8), L.OutView(0, 0, 0, 0)
    E_NULL, E_SHAPE = -1, -2
    conv = lambda **k: ctypes.byref(L.ConvArgs(**{**dict(x=v, weight=4096, bias=4096, type=0, silu=1, N=2, H=1, L=5, D=8, K=4), **k}))
    assert lib.fwp_conv_fwd(None, p, out, None) == E_NULL
    assert lib.fwp_conv_fwd(conv(x=null), p, out, None) == E_NULL
    assert lib.fwp_conv_fwd(conv(weight=0), p, out, None) == E_NULL
    assert lib.fwp_conv_fwd(conv(), p, none, None) == E_NULL
    for bad in (dict(type=3), dict(N=0), dict(H=0), dict(L=0), dict(D=0), dict(K=0), dict(K=9), dict(N=1 << 20, H=1 << 12)):
        assert lib.fwp_conv_fwd(conv(**bad), p, out, None) == E_SHAPE, bad
    assert lib.fwp_conv_fwd(conv(x=L.View(4098, 64, 32, 8)), p, out, None) == E_NULL          # half an element
    assert lib.fwp_conv_bwd(conv(), p, v, out, p, None, p, None) == E_NULL                     # one of the parameters' gradients
    assert lib.fwp_conv_bwd(conv(), p, v, out, p, p, None, None) == E_NULL
    assert lib.fwp_conv_workspace(2, 1, 5, 8, 9) == E_SHAPE and lib.fwp_conv_workspace(2, 1, 5, 8, 4) > 0
    scan = lambda **k: ctypes.byref(L.ScanArgs(**{**dict(q=v, k=v, v=v, delta=v, A=4096, type=2, N=2, H=1, L=5, E=16, M=8), **k}))
    assert lib.fwp_scan_fwd(scan(q=null), p, out, p, p, None) == E_NULL
    assert lib.fwp_scan_fwd(scan(A=0), p, out, p, p, None) == E_NULL
    assert lib.fwp_scan_workspace(2, 1, 5, 16, 8, 0) == 0 and lib.fwp_scan_workspace(1, 1, 8192, 16, 8, 0) > 0
    assert lib.fwp_scan_fwd(scan(L=8192), p, out, p, None, None) == E_NULL                     # no workspace for its segments
    for bad in (dict(E=65), dict(E=0), dict(M=0), dict(L=0), dict(type=-1)):
        assert lib.fwp_scan_fwd(scan(**bad), p, out, p, p, None) == E_SHAPE, bad
    assert lib.fwp_scan_bwd(scan(), None, v, out, out, out, out, none, p, p, p, p, None) == E_NULL
    assert lib.fwp_scan_bwd(scan(z=v), p, v, out, out, out, out, none, p, p, p, p, None) == E_NULL      # a gate without room for its gradient
    assert lib.fwp_scan_workspace(2, 1, 5, 65, 8, 0) == E_SHAPE and lib.fwp_scan_saved_floats(2, 1, 0, 16, 8) == E_SHAPE
    norm = lambda **k: ctypes.byref(L.NormArgs(**{**dict(y=4096, x=4096, before_weight=4096, type=1, stream_type=1, rows=4, cols=8), **k}))
    assert lib.fwp_residual_norm_fwd(norm(y=0), p, p, None, None) == E_NULL
    assert lib.fwp_residual_norm_fwd(norm(), p, None, None, None) == E_NULL                    # nowhere to put n
    assert lib.fwp_residual_norm_fwd(norm(before_weight=0), p, p, None, None) == E_NULL
    assert lib.fwp_residual_norm_fwd(norm(after_bias=4096), p, p, None, None) == E_NULL
    for bad in (dict(cols=8193), dict(cols=0), dict(rows=0), dict(type=5), dict(stream_type=2), dict(act=3)):
        assert lib.fwp_residual_norm_fwd(norm(**bad), p, p, None, None) == E_SHAPE, bad
    assert lib.fwp_residual_norm_bwd(norm(), None, p, p, ctypes.byref(L.NormGrads(gy=4096, gx=4096)), p, None) == E_NULL
    assert lib.fwp_residual_norm_workspace(4, 8193) == E_SHAPE
    # 2^32 threads are more than a launch has: 256 or 512 to a sequence (or four rows), 32 numbers of gq and gk to a step
    assert lib.fwp_conv_fwd(conv(N=1 << 24, L=1), p, out, None) == E_SHAPE
    assert lib.fwp_conv_bwd(conv(N=1 << 24), p, v, out, p, p, p, None) == E_SHAPE
    assert lib.fwp_scan_fwd(scan(N=1 << 24, L=1), p, out, None, None, None) == E_SHAPE
    assert lib.fwp_scan_fwd(scan(N=1 << 23), p, out, p, p, None) == E_SHAPE
    assert lib.fwp_scan_bwd(scan(N=1 << 15, L=1 << 13), p, v, out, out, out, out, none, p, p, p, p, None) == E_SHAPE
    assert lib.fwp_residual_norm_fwd(norm(rows=1 << 26), p, p, None, None) == E_SHAPE


def test_formulas_against_differences():
    """The gradients that the kernels' are compared with are the derivatives of the formulas: autograd of the forward formula, and
    central differences along a random direction."""
    torch.manual_seed(0)
    N, H, L, E, M, K = 2, 2, 6, 3, 4, 3
    d = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)
    n = torch.tensor([6, 4])
    x, w, b, st, gy = d(N, H, L, M), d(H, M, K), d(H, M), torch.randn(N, H, K - 1, M, dtype=torch.float64), torch.randn(N, H, L, M, dtype=torch.float64)
    y, _ = F.conv(x, w, b, st, True, n)
    want = torch.autograd.grad(y, [x, w, b], gy)
    with torch.no_grad():
        got = F.conv(x, w, b, st, True, n, gy)[2:]
    assert all(torch.allclose(a, c, rtol=1e-10, atol=1e-12) for a, c in zip(got, want))
    leaves = [d(N, H, L, E), d(N, H, L, E), d(N, H, L, M), d(N, H, L, M), d(H, E, M), d(H, M), d(N, H, L, M), d(H, M)]
    W = torch.randn(N, H, E, M, dtype=torch.float64)

    def out(q, k, v, delta, A, D, z, bias, go=None):
        return F.scan(q, k, v, delta, -A * A, W, D, z, bias, True, n, go)

    o = out(*leaves)[0]
    want = list(torch.autograd.grad(o, leaves, gy))
    with torch.no_grad():
        got = list(out(*leaves, go=gy)[2:])
        got[4] = -2 * leaves[4] * got[4]
        assert all(torch.allclose(a, c, rtol=1e-9, atol=1e-11) for a, c in zip(got, want))
        for i, t in enumerate(leaves):
            v, h = torch.randn_like(t), 1e-5
            plus, minus = (out(*leaves[:i], t + s * h * v, *leaves[i + 1:])[0] for s in (1, -1))
            assert abs(float(((plus - minus) / (2 * h) * gy).sum() - (got[i] * v).sum())) <= 1e-6 * (1 + float(got[i].abs().sum()))
