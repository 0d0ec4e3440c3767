"""The decayed sum rule's layer, decoder layer and a language model made of them: the block as a whole against the same block from the formulas in 64 bits, prompts and tokens
that go on from one another, padded batches, autocast, half precision.

Tolerance of the whole block: its result passes the sum (2 E + 192 + L / 8 roundings of 2^-24), the products (sums of up to 128 terms, 160 roundings) and norms (128) one after
the other, each against the size of its terms; the terms of a norm's row are sqrt(cols) at most, those of a product of its rows likewise, and the results are of
size one.  64 (L + 800) roundings of the result's largest element bound all of it."""
import copy

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import decay_formulas as F
from scan_formulas import residual_norm


def mixer(layer, h, lengths=None):
    """DecayedSumLayer from the formulas, in the parameters' type; sums over all pairs of steps"""
    T, B, _ = h.shape
    H, D = layer.n_head, layer.d_head
    x = torch.nn.functional.linear(h, layer.in_net.weight, layer.in_net.bias)
    rows = lambda i: x[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)).permute(1, 2, 0, 3)
    logit = layer.decay_logit
    logit = (logit + x[..., 4 * H * D:]).permute(1, 2, 0) if layer.token_decay else logit[None, :, None].expand(B, H, T)
    live = F.alive(lengths, B, T)
    f = F.frequencies(D)
    q, k = (F.rotary(rows(i), f, lengths=lengths) for i in (0, 1))
    b = torch.where(live[..., 0], torch.nn.functional.logsigmoid(logit), 0.0).cumsum(-1)
    apart = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -float("inf")))
    o = ((q @ k.transpose(2, 3)) * apart) @ torch.where(live, rows(2), 0.0) * D ** -0.5
    o = torch.where(live, o, 0.0).permute(2, 0, 1, 3).reshape(T, B, H * D)
    o = F.group_norm(o, H, layer.norm_weight, layer.norm_bias, x[..., 3 * H * D:4 * H * D], activation="silu")
    return torch.nn.functional.linear(o, layer.o_net.weight, layer.o_net.bias)


def decoder(m, h, lengths=None):
    norm = lambda n, t: torch.nn.functional.layer_norm(t, t.shape[-1:], n.weight, n.bias, n.eps)
    a = mixer(m.dec_attn, norm(m.norm_in, h), lengths)
    r, n = residual_norm(a, h, m.norm_attn.weight, m.norm_attn.bias, None, m.scale_attn, m.norm_mid.weight, m.norm_mid.bias)
    f = m.ff[3](torch.relu(m.ff[0](n)))
    return residual_norm(f, r, m.norm_ff.weight, m.norm_ff.bias, None, m.scale_ff)[0]


def build(fwp, d=48, heads=3, **more):
    torch.manual_seed(1)
    m = fwp.DecayedSumDecoderLayer(heads, d, d // heads, 2 * d, **more)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return m


@pytest.mark.parametrize("T,B,ragged,token_decay", [(1, 2, False, False), (37, 3, False, True), (150, 2, True, True), (70, 2, False, False)])
def test_the_block_and_its_gradients(fwp, T, B, ragged, token_decay):
    m = build(fwp, token_decay=token_decay)
    ref = copy.deepcopy(m).double()
    h, go = torch.randn(T, B, 48), torch.randn(T, B, 48)
    n = torch.tensor([T, T // 3]) if ragged else None
    hd = h.double().requires_grad_()
    want = decoder(ref, hd, n)
    want_grads = torch.autograd.grad(want, [hd] + list(ref.parameters()), go.double())
    m, hg = m.cuda(), h.cuda().requires_grad_()
    got = m(hg, lengths=None if n is None else n.cuda())
    grads = torch.autograd.grad(got, [hg] + list(m.parameters()), go.cuda())
    tol = 64 * (T + 800) * F.EPS32
    for name, a, b in zip(["out", "h"] + [k for k, _ in m.named_parameters()], [got, *grads], [want, *want_grads]):
        scale = float(b.detach().abs().max()) + (1e-3 if name in ("out", "h") else 1e-3 * (T * B) ** 0.5)
        assert float((F.double(a) - b).abs().max()) <= tol * scale, name


@pytest.mark.parametrize("token_decay", [False, True])
@pytest.mark.parametrize("cuts", [[0, 1, 2, 40, 64, 90], list(range(91))])
def test_a_prompt_and_its_tokens(fwp, cuts, token_decay):
    m, h = build(fwp, token_decay=token_decay).cuda(), torch.randn(90, 3, 48).cuda()
    with torch.no_grad():
        whole, (W, steps) = m(h, carry_over_fast_weight=True)
        mems, parts = None, []
        for a, b in zip(cuts, cuts[1:]):
            out, mems = m(h[a:b], mems=mems, carry_over_fast_weight=True)
            parts.append(out)
    tol = 64 * (90 + 800) * F.EPS32
    assert float((torch.cat(parts) - whole).abs().max()) <= tol * float(whole.abs().max())
    assert float((mems[0] - W).abs().max()) <= tol * float(W.abs().max()) and torch.equal(mems[1], steps) and int(steps[0]) == 90


def test_a_padded_batch_goes_on(fwp):
    """Prompts of different lengths, then tokens of each, against every sequence by itself"""
    m, h = build(fwp, token_decay=True).cuda(), torch.randn(40, 3, 48).cuda()
    n = torch.tensor([40, 7, 23]).cuda()
    token = torch.randn(1, 3, 48).cuda()
    with torch.no_grad():
        out, mems = m(h, carry_over_fast_weight=True, lengths=n)
        after, mems = m(token, mems=mems, carry_over_fast_weight=True)
        for i, L in enumerate(n.tolist()):
            alone, own = m(h[:L, i:i + 1], carry_over_fast_weight=True)
            next_, own = m(token[:, i:i + 1], mems=own, carry_over_fast_weight=True)
            tol = 64 * (40 + 800) * F.EPS32
            assert float((out[:L, i:i + 1] - alone).abs().max()) <= tol * float(alone.abs().max())
            assert float((after[:, i:i + 1] - next_).abs().max()) <= tol * float(next_.abs().max()) and int(mems[1][i]) == L + 1


@pytest.mark.parametrize("token_decay", [False, True])
def test_autocast_and_half_precision(fwp, token_decay):
    m, h = build(fwp, token_decay=token_decay).cuda(), torch.randn(50, 2, 48).cuda()
    want = m(h)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(h)
    # a dozen roundings to bf16 on the way
    assert float((got.float() - want).norm()) <= 16 * 2.0 ** -8 * float(want.norm())
    mixer = copy.deepcopy(m.dec_attn).bfloat16()
    out, (W, steps) = mixer(h.bfloat16(), carry_over_fast_weight=True)
    assert out.dtype is torch.bfloat16 and W.dtype is torch.float32 and mixer._frequencies.dtype is torch.float64
    assert float((out.float() - m.dec_attn(h)).norm()) <= 16 * 2.0 ** -8 * float(out.float().norm())


@pytest.mark.parametrize("token_decay", [False, True])
def test_a_language_model_of_them(fwp, token_decay):
    torch.manual_seed(0)
    import functools
    layer = functools.partial(fwp.DecayedSumDecoderLayer, token_decay=token_decay)
    lm = fwp.DeltaNetLM(97, 2, 4, 64, 16, 128, decoder_layer=layer).cuda()
    data, target = torch.randint(0, 97, (70, 3)).cuda(), torch.randint(0, 97, (70, 3)).cuda()
    loss = lm(data, target)[0]
    loss.mean().backward()
    assert loss.shape == (70, 3) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in lm.parameters())
    with torch.no_grad():
        hid, mems = lm.hidden(data, carry_over_fast_weight=True)
        again, mems = lm.hidden(data[:1], mems, carry_over_fast_weight=True)
    assert torch.isfinite(again).all() and int(mems[0][1][0]) == 71


@pytest.mark.parametrize("token_decay", [False, True])
def test_training_after_inference_mode(fwp, token_decay):
    """What a call under inference mode leaves, in the layer and as its state, is no obstacle to training"""
    layer = build(fwp, token_decay=token_decay).cuda()
    h = torch.randn(20, 2, 48).cuda()
    with torch.inference_mode():
        first, mems = layer(h[:12], carry_over_fast_weight=True)
    y, _ = layer(h[12:], mems=mems, carry_over_fast_weight=True)
    grads = torch.autograd.grad(y.square().sum(), list(layer.parameters()))
    assert all(torch.isfinite(g).all() for g in grads)
    with torch.no_grad():
        want, state = layer(h[:12], carry_over_fast_weight=True)
        assert torch.equal(first, want)
    z, _ = layer(h[12:], mems=state, carry_over_fast_weight=True)
    assert torch.equal(y, z)
    for a, b in zip(grads, torch.autograd.grad(z.square().sum(), list(layer.parameters()))):
        assert torch.equal(a, b)
