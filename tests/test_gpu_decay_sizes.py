"""The decayed sum rule at every width its tiles come in, whole and cut, in several segments and slices; values that are not finite; calls from several threads and
on several streams; tensors that cannot be kept.  Tolerances as in test_gpu_decay.py."""
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F
from test_gpu_decay import TYPES, check, decays, lengths_of, randn, rows, sum_formulas, sum_inputs


def both_ways(fwp, g, dtype, N, H, G, L, E, M, layout, decay, ragged, scale=0.3):
    t, W = sum_inputs(g, dtype, N, H, G, L, E, M, layout, True, decay)
    n = lengths_of(N, L, g) if ragged else None
    go = rows(g, dtype, N, H, L, M, "steps")
    want = sum_formulas(t, W, scale, n, go)
    sizes = list(zip(*[sum_formulas(t, W, scale, n, go, absolute=True, **x) for x in ({}, {"halved": True})]))
    leaves = {k: x.detach().requires_grad_() for k, x in t.items()}
    out = fwp.decayed_sum(**leaves, W=W, scale=scale, lengths=n)
    grads = torch.autograd.grad(out, list(leaves.values()), go)
    forward, backward = 2 * E + 192 + L // 8, 4 * (E + M) + 512 + L // 4
    check(out, want[0], sizes[0], forward, "out", dtype)
    check(W, want[1], sizes[1], forward, "W", torch.float32)
    for i, name in enumerate(["Q", "K", "V", "log_decay"]):
        extra = N * L if name == "log_decay" and t[name].dim() == 1 else ([H // x for x in G] + [1])[i]
        check(grads[i], want[2 + i], sizes[2 + i], backward + extra, "gradient of " + name, torch.float32 if i == 3 else dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [32, 64, 128, 3, 40, 127])
@pytest.mark.parametrize("M", [32, 64, 128, 256, 2, 57, 65, 190])
def test_every_width(fwp, E, M, dtype):
    g = torch.Generator().manual_seed(1000 * E + M)
    both_ways(fwp, g, dtype, 2, 2, (2, 1, 2) if E % 2 else (2, 2, 1), 150, E, M, "steps", "token" if M % 2 else "head", E == 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,G,L,E,M,decay", [(5, 2, (1, 1, 2), 500, 32, 32, "token"), (6, 1, (1, 1, 1), 641, 64, 64, "head"), (3, 4, (1, 2, 4), 400, 16, 130, "strong"),
                                               (4, 2, (2, 2, 1), 257, 128, 100, "head")])
def test_padded_batches_in_segments(fwp, N, H, G, L, E, M, decay, dtype):
    g = torch.Generator().manual_seed(L)
    both_ways(fwp, g, dtype, N, H, G, L, E, M, "steps", decay, True)


# ------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,M,L", [(32, 32, 100), (20, 40, 90), (64, 64, 300), (128, 130, 200), (48, 100, 5), (16, 16, 1500)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_steps_before_a_value_that_is_not_finite_do_not_see_it(fwp, E, M, L, bad, dtype):
    g = torch.Generator().manual_seed(E + L)
    t, _ = sum_inputs(g, dtype, 2, 2, (2, 2, 2), L, E, M, "steps", False, "token")
    run = lambda **x: (lambda W: (fwp.decayed_sum(**{**t, **x}, W=W), W))(torch.zeros(2, 2, E, M).cuda())
    with torch.no_grad():
        out, W = run()
        for at in {0, L // 3, min(L - 1, 63), min(L - 1, 64), L - 1}:
            def spoiled(name, *where):
                x = t[name].clone()
                x[(1, 1, at, *where)] = bad
                return run(**{name: x})
            # a value: its own column, from its step on
            m = M // 2
            o, w = spoiled("V", m)
            others = torch.arange(M).cuda() != m
            assert torch.equal(o[0], out[0]) and torch.equal(o[1, 0], out[1, 0]) and torch.equal(o[1, 1, :at], out[1, 1, :at])
            assert torch.equal(o[1, 1][:, others], out[1, 1][:, others]) and not torch.isfinite(o[1, 1, at:, m]).any()
            assert torch.equal(w[1, 1][:, others], W[1, 1][:, others]) and not torch.isfinite(w[1, 1, :, m]).any()
            # a key: every column, from its step on, and its own row of the state
            o, w = spoiled("K", E - 1)
            assert torch.equal(o[1, 1, :at], out[1, 1, :at]) and not torch.isfinite(o[1, 1, at:]).any()
            assert torch.equal(w[1, 1, :E - 1], W[1, 1, :E - 1]) and not torch.isfinite(w[1, 1, E - 1]).any()
            # a query: its own step
            o, w = spoiled("Q", 0)
            rest = torch.arange(L).cuda() != at
            assert torch.equal(o[1, 1][rest], out[1, 1][rest]) and not torch.isfinite(o[1, 1, at]).any() and torch.equal(w, W)
            if bad != bad:
                o, w = spoiled("log_decay")
                assert torch.equal(o[1, 1, :at], out[1, 1, :at]) and (at == 0 or not torch.isfinite(o[1, 1, at:]).any())


# ------------------------------------------------------------------ streams, threads, inference mode

def test_threads_and_streams_at_once(fwp):
    """Four threads, each on a stream of its own, forward and backward, against the same calls one after another"""
    g = torch.Generator().manual_seed(4)
    calls = []
    for i in range(4):
        t, W = sum_inputs(g, torch.bfloat16, 2, 4, (1, 2, 4), 300 + 40 * i, 64, 64 + 32 * (i % 2), "steps", True, "token")
        calls.append((t, W, rows(g, torch.bfloat16, 2, 4, 300 + 40 * i, 64 + 32 * (i % 2))))

    def run(t, W, go):
        W = W.clone()
        leaves = {k: x.detach().requires_grad_() for k, x in t.items()}
        out = fwp.decayed_sum(**leaves, W=W)
        return out.detach(), W, *torch.autograd.grad(out, list(leaves.values()), go)
    want = [run(*c) for c in calls]
    torch.cuda.synchronize()
    got, errors = [[] for _ in calls], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(3):
                    got[i].append(run(*calls[i]))
            s.synchronize()
        except Exception as e:      # a failure in a thread would pass otherwise
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not errors
    for i, w in enumerate(want):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, w)), i


@pytest.mark.parametrize("name", ["Q", "K", "V", "log_decay", "lengths"])
def test_refused_with_the_state_as_it_was(fwp, name):
    g = torch.Generator().manual_seed(5)
    t, W = sum_inputs(g, torch.float32, 2, 2, (2, 2, 2), 9, 8, 8, "plain", True, "token")
    t["lengths"] = torch.tensor([9, 4]).cuda()
    with torch.inference_mode():
        t[name] = t[name].clone()
    leaf = "Q" if name != "Q" else "K"
    t[leaf] = t[leaf].requires_grad_()
    before = W.clone()
    with pytest.raises(fwp._lib.FwpError, match="inference"):
        fwp.decayed_sum(**t, W=W)
    assert torch.equal(W, before)
    with torch.no_grad():
        fwp.decayed_sum(**t, W=W)
    assert not torch.equal(W, before)


@pytest.mark.parametrize("op", ["rotary", "group_norm"])
def test_others_refuse_too(fwp, op):
    x = torch.randn(2, 2, 9, 8).cuda()
    with torch.inference_mode():
        w = torch.ones(8).cuda()
        f = F.frequencies(8).cuda()
    with pytest.raises(fwp._lib.FwpError, match="inference"):
        fwp.rotary(x.clone().requires_grad_(), None, f) if op == "rotary" else fwp.group_norm(x.clone().requires_grad_(), 2, w)


# ------------------------------------------------------------------ calls that the documentation allows

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,pairs", [(32, 16), (37, 12)])
def test_rotary_in_place(fwp, D, pairs, interleaved, dtype):
    """The C entry may write the rows that it reads"""
    import ctypes
    L = fwp._lib
    g = torch.Generator().manual_seed(D)
    q, k, f = rows(g, dtype, 2, 9, 33, D), rows(g, dtype, 2, 3, 33, D), F.frequencies(2 * pairs).cuda()
    want = fwp.rotary(q, k, f, interleaved=interleaved, scale=0.7)
    view = lambda t, kind: kind(t.data_ptr(), *t.stride()[:3])
    a = L.RotaryArgs(q=view(q, L.View), k=view(k, L.View), frequencies=f.data_ptr(), scale=0.7, type=TYPES.index(dtype), interleaved=interleaved, N=2, HQ=9, HK=3, L=33, D=D, pairs=pairs)
    assert L.lib().fwp_rotary(ctypes.byref(a), view(q, L.OutView), view(k, L.OutView), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_of_any_dimensions_and_broadcast_rows(fwp, dtype):
    g = torch.Generator().manual_seed(2)
    x, w = randn(g, 3, 4, 5, 48).to(dtype).cuda(), randn(g, 48).cuda()
    want = fwp.group_norm(x, 6, w, activation="silu")
    assert torch.equal(fwp.group_norm(x.view(60, 48), 6, w, activation="silu").view_as(x), want)
    assert torch.equal(fwp.group_norm(x[1, 2, 3], 6, w, activation="silu"), want[1, 2, 3])
    one = randn(g, 1, 48).to(dtype).cuda().requires_grad_()
    flat = x.view(60, 48)
    y = fwp.group_norm(flat, 6, w, gate=one.expand(60, 48), activation="sigmoid")
    dense = one.detach().expand(60, 48).contiguous().requires_grad_()
    z = fwp.group_norm(flat, 6, w, gate=dense, activation="sigmoid")
    assert torch.equal(y, z)
    a, b = torch.autograd.grad(y, one, flat)[0], torch.autograd.grad(z, dense, flat)[0]
    # 60 terms added in one order or another, in fp32 or more, and rounded once
    exact = F.double(b).sum(0, keepdim=True)
    assert float((F.double(a) - exact).abs().max()) <= 60 * F.EPS32 * float(F.double(b).abs().sum(0).max()) + F.half_step(dtype) * float(exact.abs().max())


def test_broadcast_queries_and_decays(fwp):
    g = torch.Generator().manual_seed(3)
    q, d = randn(g, 1, 1, 70, 16).cuda().requires_grad_(), decays(g, 1, 1, 70, "token").requires_grad_()
    k, v, go = rows(g, torch.float32, 3, 4, 70, 16), rows(g, torch.float32, 3, 4, 70, 20), rows(g, torch.float32, 3, 4, 70, 20)
    out = fwp.decayed_sum(q.expand(3, 4, 70, 16), k, v, d.expand(3, 4, 70))
    grads = torch.autograd.grad(out, (q, d), go)
    full = [t.detach().expand(3, 4, *t.shape[2:]).contiguous().requires_grad_() for t in (q, d)]
    same = fwp.decayed_sum(full[0], k, v, full[1])
    assert torch.equal(out, same)
    for a, b in zip(grads, torch.autograd.grad(same, full, go)):
        b = F.double(b)
        assert float((F.double(a) - b.sum((0, 1), keepdim=True)).abs().max()) <= 12 * F.EPS32 * float(b.abs().sum((0, 1)).max())
