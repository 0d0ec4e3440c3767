"""The selective scan's layer, decoder layer and a language model made of them: the block as a whole against the same block from the formulas in 64 bits,
prompts and tokens that go on from one another, padded batches, autocast.

Tolerance of the whole block: its result passes the scan ((4 L + E + 64) roundings of 2^-24), the products (sums of up to 128 terms, 160
roundings) and norms (128) one after the other, each against the size of its terms; the terms of a norm's row are sqrt(cols) at most, those
of a product of its rows likewise, and the results are of size one.  64 (4 L + 400) roundings of the result's largest element bound all of it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import scan_formulas as F


def mixer(layer, h, lengths=None):
    """SelectiveScanLayer from the formulas, in the parameters' type"""
    C, E = layer.channels, layer.n_state
    rows = lambda t: t[:, :, None].permute(1, 2, 0, 3)
    steps = lambda t: t.permute(2, 0, 1, 3).reshape(h.shape[0], h.shape[1], -1)
    lin = torch.nn.functional.linear
    x, z = (rows(t) for t in lin(h, layer.in_net.weight, layer.in_net.bias).split(C, -1))
    v, _ = F.conv(x, layer.conv_weight, layer.conv_bias, None, True, lengths)
    rank, q, k = lin(steps(v), layer.step_net.weight, layer.step_net.bias).split((layer.rank, E, E), -1)
    out, _ = F.scan(rows(q), rows(k), v, rows(lin(rank, layer.delta_net.weight)), -torch.exp(layer.log_decay), None, layer.skip, z,
                    layer.delta_bias, True, lengths)
    return lin(steps(out), layer.o_net.weight, layer.o_net.bias)


def decoder(m, h, lengths=None):
    norm = lambda n, t: torch.nn.functional.layer_norm(t, t.shape[-1:], n.weight, n.bias, n.eps)
    a = mixer(m.dec_attn, norm(m.norm_in, h), lengths)
    r, n = F.residual_norm(a, h, m.norm_attn.weight, m.norm_attn.bias, None, m.scale_attn, m.norm_mid.weight, m.norm_mid.bias)
    f = m.ff[3](torch.relu(m.ff[0](n)))
    return F.residual_norm(f, r, m.norm_ff.weight, m.norm_ff.bias, None, m.scale_ff)[0]


def build(fwp, d=48, **more):
    torch.manual_seed(1)
    m = fwp.SelectiveScanDecoderLayer(4, d, d // 4, 2 * d, **more)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return m


@pytest.mark.parametrize("T,B,ragged", [(1, 2, False), (37, 3, False), (150, 2, True)])
def test_the_block_and_its_gradients(fwp, T, B, ragged):
    import copy
    m = build(fwp)
    ref = copy.deepcopy(m).double()
    h = torch.randn(T, B, 48)
    go = torch.randn(T, B, 48)
    n = torch.tensor([T, T // 3]) if ragged else None
    hd = h.double().requires_grad_()
    want = decoder(ref, hd, n)
    want_grads = torch.autograd.grad(want, [hd] + list(ref.parameters()), go.double())
    m, hg = m.cuda(), h.cuda().requires_grad_()
    got = m(hg, lengths=None if n is None else n.cuda())
    grads = torch.autograd.grad(got, [hg] + list(m.parameters()), go.cuda())
    tol = 64 * (4 * T + 400) * F.EPS32
    for name, a, b in zip(["out", "h"] + [k for k, _ in m.named_parameters()], [got, *grads], [want, *want_grads]):
        # a parameter's gradient adds up the tokens' shares
        scale = float(b.detach().abs().max()) + (1e-3 if name in ("out", "h") else 1e-3 * (T * B) ** 0.5)
        assert float((F.double(a) - b).abs().max()) <= tol * scale, name


def test_gradients_against_differences(fwp):
    m, h, go = build(fwp).cuda(), torch.randn(20, 2, 48).cuda(), torch.randn(20, 2, 48).cuda()
    params = list(m.parameters())
    grads = torch.autograd.grad(m(h), params, go)
    import copy
    ref = copy.deepcopy(m).cpu().double()
    for (name, p), g in zip(ref.named_parameters(), grads):
        v, step = torch.randn_like(p), 1e-5
        with torch.no_grad():
            p.add_(step * v)
            up = decoder(ref, h.cpu().double())
            p.sub_(2 * step * v)
            down = decoder(ref, h.cpu().double())
            p.add_(step * v)
        slope = float(((up - down) / (2 * step) * go.cpu().double()).sum())
        # the difference is off by step^2 of the third derivative, the gradient as above
        assert abs(slope - float((F.double(g) * v).sum())) <= 3e-4 * float((F.double(g) * v).norm()) * v.numel() ** 0.25 + 1e-4, name


@pytest.mark.parametrize("cuts", [[0, 1, 2, 40, 64, 90], list(range(91))])
def test_a_prompt_and_its_tokens(fwp, cuts):
    m, h = build(fwp).cuda(), torch.randn(90, 3, 48).cuda()
    with torch.no_grad():
        whole, (W, state) = m(h, carry_over_fast_weight=True)
        plain = m(h)
        assert torch.equal(plain, whole)
        mems, outs = None, []
        for a, b in zip(cuts, cuts[1:]):
            out, mems = m(h[a:b], mems=mems, carry_over_fast_weight=True)
            outs.append(out)
    tol = 64 * (4 * 90 + 400) * F.EPS32
    for a, b in ((torch.cat(outs), whole), (mems[0], W), (mems[1], state)):
        assert float((a - b).abs().max()) <= tol * (1 + float(b.abs().max()))


def test_a_smaller_batch_and_mems_that_are_not_carried(fwp):
    m, h = build(fwp).cuda(), torch.randn(5, 3, 48).cuda()
    with torch.no_grad():
        _, mems = m(h, carry_over_fast_weight=True)
        kept = [t.clone() for t in mems]
        out, (W, _) = m(h[:, :2], mems=mems, carry_over_fast_weight=True)
        assert out.shape == (5, 2, 48) and W.shape[0] == 2 and all(torch.equal(a, b) for a, b in zip(mems, kept))
    with pytest.raises(ValueError, match="carry_over_fast_weight"):
        m(h, mems=mems)
    with pytest.raises(ValueError, match="own operator"):
        fwp.SelectiveScanDecoderLayer(4, 48, 12, 96, fast_weight_op=fwp.fast_weight_delta)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_under_autocast(fwp, dtype):
    m, h = build(fwp).cuda(), torch.randn(60, 2, 48).cuda()
    want = m(h)
    with torch.autocast("cuda", dtype):
        got = m(h)
        got.float().square().mean().backward()
    # about sixteen roundings of the narrow type lie on the way
    assert got.dtype is torch.float32 and float((got - want).norm()) <= 16 * F.half_step(dtype) * float(want.norm())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


def test_a_language_model_of_such_layers(fwp):
    torch.manual_seed(2)
    lm = fwp.DeltaNetLM(100, 2, 4, 64, 16, 128, decoder_layer=fwp.SelectiveScanDecoderLayer).cuda()
    data, target = torch.randint(100, (30, 3)).cuda(), torch.randint(100, (30, 3)).cuda()
    loss, = lm(data, target)
    loss.mean().backward()
    assert loss.shape == (30, 3) and torch.isfinite(loss).all()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in lm.parameters())
    with torch.no_grad():
        whole, mems = lm.hidden(data, carry_over_fast_weight=True)
        assert len(mems) == 2
        # a token after the prompt, as decoding goes: positions count down to the newest token, so a call's are its own
        one, more = lm.hidden(data[-1:], mems, carry_over_fast_weight=True)
    assert one.shape == (1, 3, 64) and not torch.equal(more[0][0], mems[0][0])
