"""The selective state space block's variants that are chosen by size: the convolution's longer runs, the single step of many channels, segments at every
width of state, and the norms' adjoint with more rows than workgroups.  Against the same formulas in 64 bits as the small sizes, with their tolerances
(counted in test_gpu_scan.py and test_gpu_residual_norm.py) but for sums over all steps or rows, whose order is counted here."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import scan_formulas as F
import test_gpu_residual_norm as norms
import test_gpu_scan as scans

TYPES = scans.TYPES

# four channels of a row are a vector: runs are 8 steps below a million of them forward, 16 below four million, then 32; in the adjoint 16 below two million,
# then 32, and 64 from four million on beyond four taps
CONV = [  # N, L, D, K, layout, carried
    (33, 501, 250, 4, "plain", True), (67, 501, 252, 3, "steps", False), (67, 501, 250, 8, "plain", False), (129, 501, 252, 4, "steps", True),
    (129, 501, 250, 6, "slice", True), (129, 501, 252, 8, "plain", False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,L,D,K,layout,carried", CONV)
def test_long_runs(fwp, N, L, D, K, layout, carried, dtype):
    """All steps of all sequences, for the channels of the row's both ends and some between.  A parameter's gradient adds up at most 64 steps of a run, 4 runs of a
    workgroup, 17 of the 129 x 8 workgroups' sums (every 64th) and 20 of the slices: fewer than 128 roundings."""
    g = torch.Generator().manual_seed(N + D + K)
    x, gy = scans.rows(g, dtype, N, 1, L, D, layout), scans.rows(g, dtype, N, 1, L, D, "steps")
    w, b = scans.randn(g, 1, D, K).cuda(), scans.randn(g, 1, D).cuda()
    state = scans.randn(g, N, 1, K - 1, D).to(dtype).cuda() if carried else None
    n = scans.lengths_of(N, L, g)
    n[5:] = torch.where(n[5:] < L // 2, L, n[5:])      # most sequences are long
    c = [0, 1, 2, 3, 4, 7, 125, 126, 127, 128, D - 7, D - 6, D - 5, D - 4, D - 3, D - 2, D - 1]
    ref = [F.double(t) for t in (x[..., c], w[:, c], b[:, c], None if state is None else state[..., c])]
    args = dict(silu=True, lengths=n, gy=F.double(gy[..., c]))
    want, size = F.conv(*ref, **args), F.conv(*ref, **args, absolute=True)
    leaves = [x.detach().requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    y = fwp.causal_conv(*leaves, state, silu=True, lengths=n)
    gx, gw, gb = torch.autograd.grad(y, leaves, gy)
    scans.check(y[..., c], want[0], size[0] * 1.1, K + 24, "y", dtype)
    if carried:
        assert torch.equal(F.double(state[..., c]), want[1])
    scans.check(gx[..., c], want[2], size[2], 3 * K + 32, "gx", dtype)
    scans.check(gw[:, c], want[3], size[3], 3 * K + 32 + 128, "gw", torch.float32)
    scans.check(gb[:, c], want[4], size[4], 3 * K + 32 + 128, "gb", torch.float32)


STEPS = [(256, 1, 1028, 18), (64, 5, 1028, 7), (1024, 1, 256, 33), (130, 2, 1100, 64)]       # N, H, M, E: 2^18 channels in all, four of them to a lane


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,M,E", STEPS)
def test_one_step_of_many_channels(fwp, N, H, M, E, dtype):
    assert M % 4 == 0 and M >= 256 and N * H * M >= 1 << 18
    g = torch.Generator().manual_seed(M + E)
    t = scans.scan_inputs(g, dtype, N, H, 1, E, M, "slice", True, True)
    n = torch.randint(0, 2, (N,), generator=g)
    n[0], n[1], n[-1] = 1, 0, 9
    for lengths in (None, n.cuda()):
        for kept in (True, False):
            u = {**t, "W": t["W"].clone() if kept else None}
            (want, W), (size, W_size) = (scans.formulas(u, True, lengths, absolute=a) for a in (False, True))
            with torch.no_grad():
                out = fwp.selective_scan(**u, softplus=True, lengths=lengths)
                scans.check(out, want, size, 4 + E + 64, "out", dtype)
                if kept:
                    scans.check(u["W"], W, W_size, 4 + E + 64, "W", torch.float32)
                    if lengths is not None:
                        assert torch.equal(u["W"][1], t["W"][1])
                    # four bytes further on: one channel to a lane
                    odd = torch.cat([t["W"].new_zeros(1), t["W"].flatten()])[1:].view(t["W"].shape)
                    assert odd.data_ptr() % 16 == 4 and odd.is_contiguous()
                    again = fwp.selective_scan(**{**u, "W": odd}, softplus=True, lengths=lengths)
                    scans.check(again, want, size, 4 + E + 64, "out", dtype)
                    scans.check(odd, W, W_size, 4 + E + 64, "W", torch.float32)


# Beyond 32 keys states are kept every 8 steps and the passes work on 16: a segment of 72 steps ends within a tile of theirs
SEGMENTS = [  # N, H, L, E, M, layout, lengths, carried, gated
    (2, 1, 300, 24, 40, "plain", None, True, True), (1, 2, 333, 32, 70, "steps", None, False, False), (4, 1, 301, 17, 33, "slice", (301, 160, 7, 250), True, True),
    (3, 1, 1500, 27, 20, "steps", (1500, 1001, 144), True, True), (2, 1, 133, 40, 40, "plain", None, True, True), (1, 1, 133, 64, 64, "steps", None, False, True),
    (5, 1, 133, 33, 20, "slice", (133, 66, 72, 75, 0), True, True), (4, 1, 330, 64, 20, "plain", (330, 71, 150, 217), True, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,L,E,M,layout,lengths,carried,gated", SEGMENTS)
def test_segments_at_every_width_of_state(fwp, monkeypatch, N, H, L, E, M, layout, lengths, carried, gated, dtype):
    lib, waves, rows = fwp._lib.lib(), 8, 4 if E <= 32 else 8
    step = 16 if E <= 32 else 8
    whole = (M + 63) // 64 * N * H * -(-L // step) * step * waves * 2 * rows + N * H * (E + 2) * M      # what the adjoint's sums take without segments
    assert lib.fwp_scan_workspace(N, H, L, E, M, 0) > 0 and lib.fwp_scan_workspace(N, H, L, E, M, 1) > whole
    if lengths:
        monkeypatch.setattr(scans, "lengths_of", lambda N, L, g: torch.tensor(lengths).cuda())
    scans.test_scan(fwp, N, H, L, E, M, layout, lengths is not None, carried, gated, dtype)


# More rows than the adjoint's workgroups hold at once, the last pass over them in part
ROWS = [  # as test_gpu_residual_norm's
    ((9001, 200), False, "full", "sigmoid", True, 2, 2), ((5003, 255), True, "one", "silu", True, 1, 1), ((4501, 500), False, "full", "silu", True, 2, 2),
    ((1101, 800), False, "one", None, True, 2, 2), ((1030, 1999), True, "full", "sigmoid", True, 1, 1), ((601, 2560), True, "full", "silu", True, 1, 1),
    ((600, 4095), False, "full", "sigmoid", True, 2, 2), ((601, 4100), False, "full", None, True, 2, 2), ((300, 4099), True, "one", "sigmoid", True, 1, 1),
    ((530, 8192), True, "full", "silu", True, 1, 1), ((9001, 3), False, "full", "sigmoid", True, 2, 2),
]


@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shape,rms,gating,act,scaled,after,before", ROWS)
def test_more_rows_than_workgroups(fwp, monkeypatch, shape, rms, gating, act, scaled, after, before, dtype, stream):
    """A column's sum over the rows: at most three of a wave, four waves, 16 of 1024 workgroups (every 64th) and 20 of the slices, fewer than 64 roundings."""
    real = norms.check
    monkeypatch.setattr(norms, "check", lambda got, want, size, dtype, what, more=0: real(got, want, size, dtype, what, min(more, 64)))
    norms.test_rows(fwp, shape, rms, gating, act, scaled, after, before, dtype, stream)


@pytest.mark.parametrize("E", [4, 16, 40])
def test_steps_far_apart_in_place(fwp, E):
    """Steps just within what is read in place: a tile's offsets pass 2^31 bytes, a sequence's 2^32.  The same numbers as from copies, forward and backward."""
    N, L, M = 2, 41, 8
    g = torch.Generator().manual_seed(E)
    wide = torch.empty(L, (1 << 25) - 7, dtype=torch.float32, device="cuda")      # 5.5 GB
    at = wide.shape[1] - N * (3 * M + 2 * E) - 3
    block = wide[:, at:at + N * (3 * M + 2 * E)].view(L, N, 1, 3 * M + 2 * E)
    block.copy_(scans.randn(g, L, N, 1, 3 * M + 2 * E))
    views = [t.permute(1, 2, 0, 3) for t in block.split([M, M, M, E, E], -1)]
    A, go = -torch.rand(1, E, M, generator=g).cuda(), scans.randn(g, N, 1, L, M).cuda()
    seen = []
    for rows in (views, [t.contiguous() for t in views]):
        v, delta, z, q, k = (t.detach().requires_grad_() for t in rows)
        A_ = A.clone().requires_grad_()
        out = fwp.selective_scan(q, k, v, delta, A_, Z=z, softplus=True)
        seen.append([out, *torch.autograd.grad(out, [q, k, v, delta, z, A_], go)])
    assert all(torch.equal(a, b) for a, b in zip(*seen))


def test_very_many_sequences(fwp):
    """70000 of them, with the formula for every one."""
    N, L, E, M = 70000, 3, 4, 5
    g = torch.Generator().manual_seed(2)
    t = scans.scan_inputs(g, torch.float32, N, 1, L, E, M, "plain", True, True)
    go = scans.randn(g, N, 1, L, M).cuda()
    want, size = scans.formulas(t, True, None, go), scans.formulas(t, True, None, go, absolute=True)
    names = ["Q", "K", "V", "delta", "A", "D", "Z", "delta_bias"]
    for k in names:
        t[k] = t[k].detach().requires_grad_()
    out = fwp.selective_scan(**t, softplus=True)
    scans.check(out, want[0], size[0], 4 * L + E + 64, "out", torch.float32)
    scans.check(t["W"], want[1], size[1], 4 * L + E + 64, "W", torch.float32)
    # a parameter's gradient adds up every fourth of the sequences' sums: 17500, and three more
    for k, got, i in zip(names, torch.autograd.grad(out, [t[k] for k in names], go), range(2, 10)):
        scans.check(got, want[i], size[i], 8 * L + 2 * E + M + 128 + (17504 if k in ("A", "D", "delta_bias") else 0), "gradient of " + k, torch.float32)
