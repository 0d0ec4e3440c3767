"""Infinite values in the selective scan: which results are infinite, and which are none at all, is what the formula in 64 bits says, whether a sequence is
worked on in one piece or in segments."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import scan_formulas as F
import test_gpu_scan as scans

INF = float("inf")
NAMES = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias"]


def kinds(t):
    t = F.double(t)
    return torch.isposinf(t) * 1 + torch.isneginf(t) * 2 + torch.isnan(t) * 3


def same(got, want, what):
    a, b = kinds(got), kinds(want)
    assert torch.equal(a, b), (what, int((a != b).sum()), a[a != b][:5], b[a != b][:5])


def inputs(N, L, E, M, seed):
    """Steps of 0.1 and decays of 16 at most: a step's is never below exp(-1.6), a segment's far below the smallest number."""
    g = torch.Generator().manual_seed(seed)
    u = lambda *s: torch.rand(*s, generator=g).cuda() + 0.1
    return dict(Q=u(N, 1, L, E), K=u(N, 1, L, E), V=u(N, 1, L, M), delta=torch.full((N, 1, L, M), 0.1).cuda(), A=-16 * torch.rand(1, E, M, generator=g).cuda(),
                D=u(1, M), Z=u(N, 1, L, M), delta_bias=torch.zeros(1, M).cuda(), W=u(N, 1, E, M))


def both(fwp, t, go):
    """(out, W, gradients) of the operator and of the formula"""
    n = ("Q", "K", "V", "delta", "A", "W", "D", "Z", "delta_bias")
    want = F.scan(*(F.double(t[k]) for k in n), go=F.double(go))
    leaves = {k: t[k].detach().requires_grad_() for k in NAMES if t[k] is not None}
    W = None if t["W"] is None else t["W"].clone()
    out = fwp.selective_scan(**{**t, **leaves, "W": W})
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), go)))
    return (out, W, grads), (want[0], want[1], dict(zip(NAMES, (want[2], want[3], want[4], want[5], want[6], want[7], want[8], want[9]))))


@pytest.mark.parametrize("N,L,E,M", [(1, 30, 16, 64), (1, 2048, 16, 64), (2, 1500, 32, 64), (1, 700, 64, 64), (1, 1024, 8, 64)])
def test_states_that_are_infinite_in_segments(fwp, N, L, E, M):
    if L > 30:
        assert fwp._lib.lib().fwp_scan_workspace(N, 1, L, E, M, 0) > 0
    go = torch.ones(N, 1, L, M).cuda()
    for change in ("value", "state", "both signs", "gradient"):
        t = inputs(N, L, E, M, L)
        if change == "value":
            t["V"][0, 0, 10, 1] = INF
        elif change == "state":
            t["W"][0, 0, 2, 5] = INF
        elif change == "both signs":
            t["W"][0, 0, 1, 7], t["V"][0, 0, L // 2, 7] = INF, -INF
        g = go.clone()
        if change == "gradient":
            g[0, 0, L - 3, 9] = INF
        got, want = both(fwp, t, g)
        same(got[0], want[0], "out")
        same(got[1], want[1], "W")
        for k in ("V", "K", "Q", "D", "Z"):
            same(got[2][k], want[2][k], "gradient of " + k + ", " + change)


def test_an_infinite_state_that_is_forgotten_at_once_is_none(fwp):
    """exp(-inf) inf, in one piece and in segments"""
    for L in (30, 2048):
        t = inputs(1, L, 16, 64, L)
        t["A"][0, 3, 4], t["W"][0, 0, 3, 4] = -INF, INF
        with torch.no_grad():
            out = fwp.selective_scan(**t)
        assert torch.isnan(out[0, 0, :, 4]).all() and torch.isnan(t["W"][0, 0, 3, 4]) and not torch.isnan(out[0, 0, :, 5]).any()
