"""Rotary positions of padded batches in place, through the C entry: rows behind a sequence become zero whatever they held, those of a sequence are those of the call that
writes elsewhere."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F
from test_gpu_decay import TYPES, rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,H,G,L,D,pairs", [(5, 9, 3, 33, 32, 16), (5, 2, 1, 70, 37, 12), (6, 16, 4, 2100, 64, 16)])
def test_padded_batches_in_place(fwp, N, H, G, L, D, pairs, interleaved, dtype):
    lib = fwp._lib
    g = torch.Generator().manual_seed(D + L)
    n = torch.tensor([0, 1, L - 1, L, L + 7, -1])[:N]
    q, k, f = rows(g, dtype, N, H, L, D), rows(g, dtype, N, G, L, D, "steps"), F.frequencies(2 * pairs).cuda()
    live = F.alive(n, N, L).cuda()
    want = [torch.where(live, t, 0.0) for t in fwp.rotary(q, k, f, interleaved=interleaved, scale=0.7)]
    q, k, n = torch.where(live, q, float("nan")), torch.where(live, k, float("inf")), n.cuda()
    view = lambda t, kind: kind(t.data_ptr(), *t.stride()[:3])
    a = lib.RotaryArgs(q=view(q, lib.View), k=view(k, lib.View), frequencies=f.data_ptr(), lengths=n.data_ptr(), scale=0.7, type=TYPES.index(dtype),
                       interleaved=interleaved, N=N, HQ=H, HK=G, L=L, D=D, pairs=pairs)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.lib().fwp_rotary(ctypes.byref(a), view(q, lib.OutView), view(k, lib.OutView), stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
