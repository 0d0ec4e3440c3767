"""The caller of ``fast_weight_delta`` in language modelling: the Delta-Net layer and the
feed-forward block that follows it, with the module and parameter names of the reference
(language_modeling/src/utils/cuda_fast_weight_layer.py:57-188, utils/model_utils.py:15-67)
so a reference state_dict loads unchanged.  On the GPU, in fp32, a layer is HIP kernels throughout: the
fast-weight operator, the elementwise lines in front of it, and the matrix products with their biases,
ReLU and residual additions (``_fwp_torch``'s blocks).  Everything else - other data types, autocast, the CPU,
sub-modules that were replaced or carry hooks - runs on stock PyTorch around the operator.  A caller may
pass another operator (tests do, to compare against a step-by-step loop); the layer then also takes
the stock-PyTorch form.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils._device import DeviceContext

from . import _lib
from .decayed_sum import decayed_sum, group_norm, rotary, rotary_frequencies
from .fast_weight import _fwp_torch, fast_weight_delta
from .selective_scan import causal_conv, residual_norm, selective_scan


def _untouched(m, cls):
    """Is this sub-module exactly a ``cls`` (not a replacement) with its class's ``forward``, that nothing is hooked to?"""
    return type(m) is cls and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
                                   or "forward" in m.__dict__)


def _watched():
    """Does a mode see the operators that are called?  (A default device is such a mode, but changes none of them.)"""
    if torch._C._len_torch_dispatch_stack():
        return True
    return any(type(torch._C._get_function_stack_at(i)) is not DeviceContext for i in range(torch._C._len_torch_function_stack()))


def _blocks(takes, *args):
    """The C++ blocks (csrc/fwp_torch_blocks.cpp) if they apply, else ``None``.  Their function ``takes`` says so of the
    tensors: ordinary ones, fp32, on the GPU, of sizes that fit one another; here: a call outside autocast, tracing, modes and
    functional transforms."""
    if _fwp_torch is None or torch.compiler.is_compiling() or torch.jit.is_tracing() or not getattr(_fwp_torch, takes)(*args):
        return None
    if (torch.is_autocast_enabled() or _watched() or torch.nn.modules.module._has_any_global_hook()
            or torch.autograd.forward_ad._current_level >= 0 or torch._C._functorch.peek_interpreter_stack() is not None):
        return None
    return _fwp_torch


def _drops(m):
    """Does this dropout module change anything now?"""
    return m.training and m.p > 0


class Linear(nn.Linear):
    """``nn.Linear`` on the package's matrix products where they apply."""

    def forward(self, x):
        if torch.jit.is_scripting():
            return F.linear(x, self.weight, self.bias)
        else:
            return self._forward(x)

    def _forward(self, x):
        blocks = _blocks("takes_linear", x, self.weight, self.bias)
        if blocks is not None:
            return blocks.linear(x, self.weight, self.bias)
        return F.linear(x, self.weight, self.bias)


def _own(m, name):
    """A parameter of a module, or the plain tensor in its place (a replica's, a flattened parameter's), or ``None``."""
    p = m._parameters.get(name)
    return p if p is not None else m.__dict__.get(name)


def decode_parameters(layer):
    """The parameters of a :class:`DeltaNetDecoderLayer` as ``decode_layers`` takes them, or ``None`` when the layer
    is not what that function computes: a replaced or hooked sub-module, an active dropout, another operator."""
    if not (_untouched(layer, DeltaNetDecoderLayer)):
        return None
    att, ff = layer._modules.get("dec_attn"), layer._modules.get("pos_ff")
    if not (_untouched(att, DeltaNetLayer) and _untouched(ff, PositionwiseFF)) or att.fast_weight_op is not fast_weight_delta:
        return None
    a, f = att._modules, ff._modules
    net = f.get("CoreNet")
    if not (_untouched(net, nn.Sequential) and len(net._modules) == 5):
        return None
    lin1, relu, drop1, lin2, drop2 = net._modules.values()
    norms, projections = (a.get("layer_norm"), f.get("layer_norm")), (a.get("qkvb_net"), a.get("o_net"))
    for m in (*projections, lin1, lin2):
        if not _untouched(m, nn.Linear):
            return None
    for m in (a.get("drop"), drop1, drop2):
        if not _untouched(m, nn.Dropout) or _drops(m):
            return None
    for m in norms:
        if not _untouched(m, nn.LayerNorm) or m.eps != norms[0].eps:
            return None
    if not _untouched(relu, nn.ReLU) or att.pre_lnorm != ff.pre_lnorm:
        return None
    if any(_own(m, "bias") is not None for m in projections):
        return None
    params = [_own(m, "weight") for m in projections]
    for m in (norms[0], lin1, lin2, norms[1]):
        params += [_own(m, "weight"), _own(m, "bias")]
    return None if any(p is None for p in params) else params


def _layer_norm(m, x):
    """``m(x)`` for a LayerNorm over the last axis."""
    if _untouched(m, nn.LayerNorm) and len(m.normalized_shape) == 1:
        blocks = _blocks("takes_layer_norm", x, m.weight, m.bias, m.normalized_shape[0])
        if blocks is not None:
            return blocks.layer_norm(x, m.weight, m.bias, m.eps)
    return m(x)


class PositionalEmbedding(nn.Module):
    """Sinusoidal embedding of a position sequence: ``[sin | cos]`` halves, shape
    ``[len, 1, demb]`` (or ``[len, bsz, demb]``).  utils/model_utils.py:15-31."""

    def __init__(self, demb):
        super().__init__()
        self.demb = demb
        self.register_buffer("inv_freq", 10000.0 ** (-torch.arange(0.0, demb, 2.0) / demb))

    def forward(self, pos_seq, bsz=None):
        phase = pos_seq[:, None] * self.inv_freq[None, :]
        emb = torch.cat((phase.sin(), phase.cos()), dim=-1).unsqueeze(1)
        return emb if bsz is None else emb.expand(-1, bsz, -1)


class PositionwiseFF(nn.Module):
    """Linear-ReLU-Linear with residual and LayerNorm (after, or before when
    ``pre_lnorm``).  utils/model_utils.py:34-67.  The reference's ReLU works in place; on a
    ``[len, bsz, d_inner]`` input that is a view of the projection's 2-D result, and autograd then
    rebuilds the base tensor in backward (three copies and a clone of the widest activation per
    layer, 4 % of the language model's step): not in place here."""

    def __init__(self, d_model, d_inner, dropout, pre_lnorm=False):
        super().__init__()
        self.d_model, self.d_inner, self.dropout, self.pre_lnorm = d_model, d_inner, dropout, pre_lnorm
        self.CoreNet = nn.Sequential(
            nn.Linear(d_model, d_inner), nn.ReLU(), nn.Dropout(dropout),
            nn.Linear(d_inner, d_model), nn.Dropout(dropout))
        self.layer_norm = nn.LayerNorm(d_model)

    def _core(self, x, residual):
        """``residual + CoreNet(x)``"""
        net = self.CoreNet
        if (_untouched(net, nn.Sequential) and len(net) == 5 and _untouched(net[0], nn.Linear) and _untouched(net[1], nn.ReLU)
                and _untouched(net[2], nn.Dropout) and _untouched(net[3], nn.Linear) and _untouched(net[4], nn.Dropout)):
            W1, b1, W2, b2 = net[0].weight, net[0].bias, net[3].weight, net[3].bias
            blocks = _blocks("takes_feed_forward", x, W1, b1, W2, b2)
            if blocks is not None and not (_drops(net[2]) or _drops(net[4])):
                return blocks.feed_forward(x, W1, b1, W2, b2, residual)
            if blocks is not None:
                hid = net[2](blocks.linear(x, W1, b1, True))
                return residual + net[4](blocks.linear(hid, W2, b2))
        return residual + net(x)

    def forward(self, inp):
        if torch.jit.is_scripting():
            out = inp + self.CoreNet(self.layer_norm(inp) if self.pre_lnorm else inp)
            return out if self.pre_lnorm else self.layer_norm(out)
        else:
            return self._forward(inp)

    def _forward(self, inp):
        if self.pre_lnorm:
            return self._core(_layer_norm(self.layer_norm, inp), inp)
        return _layer_norm(self.layer_norm, self._core(inp, inp))


def sum_normalised_elu(x):
    """``phi(x) = (elu(x) + 1) / sum_D(elu(x) + 1)``: positive features that sum to one
    (cuda_fast_weight_layer.py:118-123)."""
    x = F.elu(x) + 1.0
    return x / x.sum(-1, keepdim=True)


class DeltaNetPrep(torch.autograd.Function):
    """``q, k, v, beta = DeltaNetPrep.apply(qkvb, n_head, d_head[, q_scale])``: the lines between the layer's
    projection and the operator (cuda_fast_weight_layer.py:108-125) as one HIP kernel each way.
    ``qkvb`` is the contiguous ``[len, bsz, n_head * (3 d_head + 1)]`` projection; the results are
    contiguous ``[bsz, n_head, len, .]``: q, k through :func:`sum_normalised_elu`, v copied, beta
    through a sigmoid.  ``q_scale`` multiplies q: the operator's output is linear in q, so the
    ``1/sqrt(d_head)`` the layer applies to that output (:155-157) can ride here for free."""

    @staticmethod
    def supported(qkvb, d_head):
        return (qkvb.is_cuda and qkvb.dtype == torch.float32 and qkvb.is_contiguous()
                and d_head in (16, 32, 64))

    @staticmethod
    def forward(ctx, qkvb, n_head, d_head, q_scale=1.0):
        _lib.require_device(qkvb)
        T, B, _ = qkvb.shape
        H, D = n_head, d_head
        f32 = dict(device=qkvb.device, dtype=torch.float32)
        q, k, v = (torch.empty((B, H, T, D), **f32) for _ in range(3))
        beta = torch.empty((B, H, T, 1), **f32)
        with _lib.on_device(qkvb):
            rc = _lib.lib().fwp_deltanet_prep_fwd(qkvb.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                  beta.data_ptr(), T, B, H, D, float(q_scale),
                                                  _lib.stream_of(qkvb))
        _lib.check(rc, "fwp_deltanet_prep_fwd")
        ctx.save_for_backward(qkvb)
        ctx.dims = (T, B, H, D, float(q_scale))
        return q, k, v, beta

    @staticmethod
    def backward(ctx, gq, gk, gv, gbeta):
        (qkvb,) = ctx.saved_tensors
        T, B, H, D, q_scale = ctx.dims
        gq, gk, gv, gbeta = (g.contiguous() for g in (gq, gk, gv, gbeta))
        gqkvb = torch.empty_like(qkvb)
        with _lib.on_device(qkvb):
            rc = _lib.lib().fwp_deltanet_prep_bwd(qkvb.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(),
                                                  gbeta.data_ptr(), gqkvb.data_ptr(), T, B, H, D, q_scale,
                                                  _lib.stream_of(qkvb))
        _lib.check(rc, "fwp_deltanet_prep_bwd")
        return gqkvb, None, None, None


class DeltaNetLayer(nn.Module):
    """Delta-rule linear-Transformer layer (the reference's
    ``CudaFastWeightLinearTransformerLayer`` with its default
    ``skip_attn_normalization=True``).

    ``h`` is ``[len, bsz, d_model]``.  One projection gives q, k, v and a scalar
    write strength per head; q and k go through :func:`sum_normalised_elu`, beta
    through a sigmoid, and the fast weight memory ``W[bsz, n_head, D, D]`` (zero, or
    ``mems[0]`` when a segment's state is carried over) is updated step by step by
    ``fast_weight_delta``.  The read-out is scaled by ``1/sqrt(D)``, projected, and
    added to the input with LayerNorm.  With ``carry_over_fast_weight`` the call
    returns ``(output, (W_final, None))``.
    """

    def __init__(self, n_head, d_model, d_head, dropout=0.0, dropatt=0.0, pre_lnorm=False,
                 layer_id=None, num_layer=None, fast_weight_op=None):
        super().__init__()
        self.n_head, self.d_model, self.d_head, self.dropout = n_head, d_model, d_head, dropout
        self.layer_id, self.num_layer = layer_id, num_layer
        self.qkvb_net = nn.Linear(d_model, n_head * (3 * d_head + 1), bias=False)
        self.drop = nn.Dropout(dropout)
        self.dropatt = nn.Dropout(dropatt)
        self.o_net = nn.Linear(n_head * d_head, d_model, bias=False)
        self.layer_norm = nn.LayerNorm(d_model)
        self.scale = 1.0 / d_head ** 0.5
        self.pre_lnorm = pre_lnorm
        self.fast_weight_op = fast_weight_op or fast_weight_delta

    def _state(self, mems, carry_over_fast_weight, bsz, h, dtype):
        """The state the operator starts from and overwrites: zeros, or a copy of what was carried over."""
        if mems is None:
            return torch.zeros(bsz, self.n_head, self.d_head, self.d_head, device=h.device, dtype=dtype)
        if not carry_over_fast_weight:
            raise ValueError("mems are only meaningful with carry_over_fast_weight=True")
        # the last batch of an epoch may be smaller than the carried state
        return mems[0][:bsz].clone()

    def forward(self, h, attn_mask=None, mems=None, carry_over_fast_weight=False):
        slen, bsz, _ = h.shape
        H, D = self.n_head, self.d_head
        x = _layer_norm(self.layer_norm, h) if self.pre_lnorm else h
        # The reference's pre-LN branch adds the normalised input back (it rebinds h, :100-104).
        residual = x

        hip_op = self.fast_weight_op is fast_weight_delta
        blocks = None
        if (hip_op and _untouched(self.qkvb_net, nn.Linear) and _untouched(self.o_net, nn.Linear)
                and self.qkvb_net.bias is None and self.o_net.bias is None and _untouched(self.drop, nn.Dropout)):
            blocks = _blocks("takes_delta_block", x, self.qkvb_net.weight, self.o_net.weight, H, D)
        if blocks is not None:
            # the block fills a state that starts at zero itself, beside its pre-step
            fresh = mems is None and getattr(self._state, "__func__", None) is _zeros_or_carried
            W = (torch.empty(bsz, H, D, D, device=h.device, dtype=torch.float32) if fresh
                 else self._state(mems, carry_over_fast_weight, bsz, h, torch.float32))
            drops = _drops(self.drop)
            out = blocks.delta_block(x, self.qkvb_net.weight, self.o_net.weight, W, H, D, self.scale, not drops, fresh)
            if drops:
                out = residual + self.drop(out)
            if not self.pre_lnorm:
                out = _layer_norm(self.layer_norm, out)
            return (out, (W.detach(), None)) if carry_over_fast_weight else out

        qkvb = self.qkvb_net(x)
        fused = hip_op and DeltaNetPrep.supported(qkvb, D)
        if fused:
            # one fused kernel each way; q carries the 1/sqrt(D) of the read-out (the operator is
            # linear in q), and the operator writes [len, bsz, H, D] storage: no pass over its output
            q, k, v, beta = DeltaNetPrep.apply(qkvb, H, D, self.scale)
        else:
            qkvb = qkvb.view(slen, bsz, H, 3 * D + 1)
            q, k, v, beta = (t.permute(1, 2, 0, 3) for t in qkvb.split((D, D, D, 1), dim=-1))
            q, k, beta = sum_normalised_elu(q), sum_normalised_elu(k), torch.sigmoid(beta)

        if hip_op:
            # half or bf16 activations (autocast, which makes some of them fp32): the operator and its state are fp32, as
            # the reference's kernel and its torch.zeros state are
            q, k, v, beta = q.float(), k.float(), v.float(), beta.float()
        W = self._state(mems, carry_over_fast_weight, bsz, h, torch.float32 if hip_op else q.dtype)

        if fused:
            out = fast_weight_delta(q, k, v, beta, W, True)          # [bsz, H, slen, D] over [slen, bsz, H, D] storage
            out = out.permute(2, 0, 1, 3).reshape(slen, bsz, H * D)  # a view
        else:
            out = self.fast_weight_op(q, k, v, beta, W)              # [bsz, H, slen, D]
            out = (self.scale * out).permute(2, 0, 1, 3).reshape(slen, bsz, H * D).to(x.dtype)
        out = residual + self.drop(self.o_net(out))
        if not self.pre_lnorm:
            out = self.layer_norm(out)
        if carry_over_fast_weight:
            return out, (W.detach(), None)
        return out


_zeros_or_carried = DeltaNetLayer._state      # as it is here, whatever replaces it later


class DeltaNetDecoderLayer(nn.Module):
    """Delta-Net layer followed by the feed-forward block (``DecoderLayer`` with
    ``attn_type=24``, model_main.py:703-775); sub-module names ``dec_attn`` and
    ``pos_ff`` as there."""

    def __init__(self, n_head, d_model, d_head, d_inner, dropout=0.0, dropatt=0.0, pre_lnorm=False,
                 layer_id=None, num_layer=None, fast_weight_op=None):
        super().__init__()
        self.dec_attn = DeltaNetLayer(n_head, d_model, d_head, dropout, dropatt, pre_lnorm,
                                      layer_id, num_layer, fast_weight_op)
        self.pos_ff = PositionwiseFF(d_model, d_inner, dropout, pre_lnorm)

    def forward(self, dec_inp, dec_attn_mask=None, mems=None, carry_over_fast_weight=False):
        out = self.dec_attn(dec_inp, attn_mask=dec_attn_mask, mems=mems,
                            carry_over_fast_weight=carry_over_fast_weight)
        if carry_over_fast_weight:
            out, new_mem = out
            return self.pos_ff(out), new_mem
        return self.pos_ff(out)


class SelectiveScanLayer(nn.Module):
    """The mixer of a selective state space block, beside :class:`DeltaNetLayer`: ``h`` is ``[len, bsz, d_model]``, one projection gives the
    values and their gate (``expand * d_model`` channels each), the values go through a :func:`causal_conv` of ``taps`` taps, another
    projection of the result gives q and k (``n_state`` each, shared by all channels) and the step sizes by way of ``rank`` numbers, and
    :func:`selective_scan` and a projection back follow.  No norm and no residual: those are the block's.

    ``mems`` is the pair (``W[bsz, 1, n_state, channels]``, the convolution's last rows ``[bsz, 1, taps - 1, channels]``); with
    ``carry_over_fast_weight`` the call returns ``(output, mems)``.  ``lengths`` (int64 ``[bsz]``) marks a padded batch.  No counterpart in the reference.
    """

    def __init__(self, d_model, n_state=16, taps=4, expand=2, rank=None, dropout=0.0):
        super().__init__()
        self.d_model, self.n_state, self.taps, self.channels = d_model, n_state, taps, expand * d_model
        self.rank = rank or -(-d_model // 16)
        self.in_net = Linear(d_model, 2 * self.channels)
        self.conv_weight = nn.Parameter(torch.empty(1, self.channels, taps))
        self.conv_bias = nn.Parameter(torch.empty(1, self.channels))
        self.step_net = Linear(self.channels, self.rank + 2 * n_state)
        self.delta_net = nn.Linear(self.rank, self.channels, bias=False)
        self.delta_bias = nn.Parameter(torch.empty(1, self.channels))
        self.log_decay = nn.Parameter(torch.empty(1, n_state, self.channels))
        self.skip = nn.Parameter(torch.empty(1, self.channels))
        self.o_net = Linear(self.channels, d_model)
        self.drop = nn.Dropout(dropout)
        self.reset_scan_parameters()

    def reset_scan_parameters(self):
        """Decays of 1 .. n_state at step size 1, step sizes spread from 0.001 to 0.1 over the channels."""
        with torch.no_grad():
            self.conv_weight.uniform_(-1, 1).mul_(self.taps ** -0.5)
            self.conv_bias.zero_()
            self.log_decay.copy_(torch.arange(1.0, self.n_state + 1, device=self.log_decay.device).log()[None, :, None].expand_as(self.log_decay))
            self.skip.fill_(1.0)
            step = torch.logspace(-3, -1, self.channels, device=self.delta_bias.device)
            self.delta_bias.copy_(step + torch.log(-torch.expm1(-step)))

    def forward(self, h, attn_mask=None, mems=None, carry_over_fast_weight=False, lengths=None):
        if mems is not None and not carry_over_fast_weight:
            raise ValueError("mems are only meaningful with carry_over_fast_weight=True")
        slen, bsz, _ = h.shape
        rows = lambda t: t.view(slen, bsz, 1, -1).permute(1, 2, 0, 3)       # [bsz, 1, slen, .], the steps outermost in memory
        steps = lambda t: t.permute(2, 0, 1, 3).reshape(slen, bsz, -1)      # and back, a view
        x, z = (rows(t) for t in self.in_net(h).split(self.channels, -1))
        if not carry_over_fast_weight:
            W = state = None
        elif mems is None:
            W = torch.zeros(bsz, 1, self.n_state, self.channels, device=h.device, dtype=torch.float32)
            state = torch.zeros(bsz, 1, self.taps - 1, self.channels, device=h.device, dtype=x.dtype)
        else:       # the last batch of an epoch may be smaller than the carried state
            W, state = mems[0][:bsz].clone(), mems[1][:bsz].to(x.dtype, copy=True)
        v = causal_conv(x, self.conv_weight, self.conv_bias, state, silu=True, lengths=lengths)
        rank, q, k = self.step_net(steps(v)).split((self.rank, self.n_state, self.n_state), -1)
        out = selective_scan(rows(q), rows(k), v, rows(self.delta_net(rank)), -torch.exp(self.log_decay), W, D=self.skip, Z=z,
                             delta_bias=self.delta_bias, softplus=True, lengths=lengths)
        out = self.drop(self.o_net(steps(out)))
        return (out, (W, state)) if carry_over_fast_weight else out


class _ResidualDecoderLayer(nn.Module):
    """A mixer and the feed-forward block behind it on a residual stream: norm, mixer, norm and scale on its output, and the same around the
    feed-forward block; :func:`residual_norm` is what lies between and behind the two, but for a norm that was replaced or hooked to, which is called."""

    def __init__(self, mixer, d_model, d_inner, dropout):
        super().__init__()
        self.dec_attn = mixer
        self.norm_in, self.norm_mid = nn.LayerNorm(d_model), nn.LayerNorm(d_model)
        self.norm_attn, self.norm_ff = nn.LayerNorm(d_model), nn.LayerNorm(d_model)
        self.scale_attn, self.scale_ff = nn.Parameter(torch.ones(d_model)), nn.Parameter(torch.ones(d_model))
        self.ff = nn.Sequential(Linear(d_model, d_inner), nn.ReLU(), nn.Dropout(dropout), Linear(d_inner, d_model), nn.Dropout(dropout))

    def forward(self, dec_inp, dec_attn_mask=None, mems=None, carry_over_fast_weight=False, lengths=None):
        out = self.dec_attn(_layer_norm(self.norm_in, dec_inp), mems=mems, carry_over_fast_weight=carry_over_fast_weight, lengths=lengths)
        out, mems = out if carry_over_fast_weight else (out, None)
        r, n = _around(out, dec_inp, self.norm_attn, self.scale_attn, self.norm_mid)
        r, _ = _around(self.ff(n), r, self.norm_ff, self.scale_ff)
        return (r, mems) if carry_over_fast_weight else r


class SelectiveScanDecoderLayer(_ResidualDecoderLayer):
    """A :class:`SelectiveScanLayer` and the feed-forward block behind it on a residual stream.  Constructor and call as
    :class:`DeltaNetDecoderLayer`'s, whose place it takes in :class:`DeltaNetLM`; heads do not count here (q and k are shared by all channels),
    ``dropatt`` has nothing to drop, and norms come before a block whatever ``pre_lnorm``."""

    def __init__(self, n_head, d_model, d_head, d_inner, dropout=0.0, dropatt=0.0, pre_lnorm=True, layer_id=None, num_layer=None,
                 fast_weight_op=None, n_state=16, taps=4):
        if fast_weight_op is not None:
            raise ValueError("a selective scan layer has its own operator")
        super().__init__(SelectiveScanLayer(d_model, n_state, taps, dropout=dropout), d_model, d_inner, dropout)


class DecayedSumLayer(nn.Module):
    """The mixer whose fast weights decay, beside :class:`DeltaNetLayer`: ``h`` is ``[len, bsz, d_model]``, one projection gives queries, keys and values of ``n_head``
    heads and a gate, :func:`rotary` turns queries and keys, :func:`decayed_sum` writes and reads the fast weights, :func:`group_norm` normalises every
    head and gates it, and a projection back follows.  No norm and no residual of the stream: those are the block's.

    A head's decay is the sigmoid of a number of its own, from memories of 32 steps upwards; with ``token_decay`` the step adds to that number.  ``mems`` is the pair
    (``W[bsz, n_head, d_head, d_head]``, the steps so far ``[bsz]``, int64); with ``carry_over_fast_weight`` the call returns ``(output, mems)``.  ``lengths`` (int64
    ``[bsz]``) marks a padded batch.  No counterpart in the reference.
    """

    def __init__(self, n_head, d_model, d_head, dropout=0.0, token_decay=False):
        super().__init__()
        if d_head % 2:
            raise ValueError("rotary positions turn pairs of channels: d_head must be even")
        self.n_head, self.d_model, self.d_head, self.token_decay = n_head, d_model, d_head, token_decay
        self.in_net = Linear(d_model, 4 * n_head * d_head + (n_head if token_decay else 0))
        self.decay_logit = nn.Parameter(torch.empty(n_head))
        self.norm_weight = nn.Parameter(torch.ones(n_head * d_head))
        self.norm_bias = nn.Parameter(torch.zeros(n_head * d_head))
        self.o_net = Linear(n_head * d_head, d_model)
        self.drop = nn.Dropout(dropout)
        # no buffer: a model in half precision keeps them in 64 bits, and one that is built without memory has them all the same
        device = self.decay_logit.device
        self._frequencies = rotary_frequencies(d_head, device="cpu" if device.type == "meta" else device)[0]
        self.reset_decay_parameters()

    def reset_decay_parameters(self):
        """Memories of 32 steps for the first head, twice as long for each one behind it, up to 4096."""
        with torch.no_grad():
            steps = torch.exp2(5.0 + torch.arange(self.n_head, device=self.decay_logit.device).clamp(max=7))
            self.decay_logit.copy_(torch.log(steps - 1))

    def forward(self, h, attn_mask=None, mems=None, carry_over_fast_weight=False, lengths=None):
        if mems is not None and not carry_over_fast_weight:
            raise ValueError("mems are only meaningful with carry_over_fast_weight=True")
        slen, bsz, _ = h.shape
        H, D = self.n_head, self.d_head
        x = self.in_net(h)
        q, k, v, gate = (x[..., i * H * D:(i + 1) * H * D] for i in range(4))
        rows = lambda t: t.unflatten(-1, (H, D)).permute(1, 2, 0, 3)        # [bsz, H, slen, D], the steps outermost in memory
        logit = self.decay_logit.float()
        if self.token_decay:
            logit = (logit + x[..., 4 * H * D:].float()).permute(1, 2, 0)
        W = position = None
        if carry_over_fast_weight and mems is None:
            W = torch.zeros(bsz, H, D, D, device=h.device, dtype=torch.float32)
            position = torch.zeros(bsz, device=h.device, dtype=torch.int64)
        elif carry_over_fast_weight:       # the last batch of an epoch may be smaller than the carried state
            W, position = mems[0][:bsz].clone(), mems[1][:bsz]
            if position.is_inference() and not torch.is_inference_mode_enabled():       # autograd keeps no tensor of inference mode
                position = position.clone()
        if self._frequencies.device != h.device:
            with torch.inference_mode(False):
                self._frequencies = self._frequencies.to(h.device)
        q, k = rotary(rows(q), rows(k), self._frequencies, positions=position, lengths=lengths)
        out = decayed_sum(q, k, rows(v), F.logsigmoid(logit), W, scale=D ** -0.5, lengths=lengths)
        out = out.permute(2, 0, 1, 3).reshape(slen, bsz, H * D)
        out = group_norm(out, H, self.norm_weight.float(), self.norm_bias.float(), gate=gate, activation="silu")
        out = self.drop(self.o_net(out))
        if not carry_over_fast_weight:
            return out
        return out, (W, position + (slen if lengths is None else lengths.clamp(0, slen)))


class DecayedSumDecoderLayer(_ResidualDecoderLayer):
    """A :class:`DecayedSumLayer` and the feed-forward block behind it on a residual stream.  Constructor and call as :class:`DeltaNetDecoderLayer`'s, whose place it
    takes in :class:`DeltaNetLM`; ``dropatt`` has nothing to drop, and norms come before a block whatever ``pre_lnorm``."""

    def __init__(self, n_head, d_model, d_head, d_inner, dropout=0.0, dropatt=0.0, pre_lnorm=True, layer_id=None, num_layer=None,
                 fast_weight_op=None, token_decay=False):
        if fast_weight_op is not None:
            raise ValueError("a decayed sum layer has its own operator")
        super().__init__(DecayedSumLayer(n_head, d_model, d_head, dropout, token_decay), d_model, d_inner, dropout)


def _fuses(norm, cols):
    """Is this norm what :func:`residual_norm` computes: a LayerNorm over the last axis with a weight, that nothing watches?"""
    return (_untouched(norm, nn.LayerNorm) and not torch.nn.modules.module._has_any_global_hook() and norm.normalized_shape == (cols,)
            and norm.weight is not None)


def _around(y, x, after, scale, before=None):
    """``r = x + scale after(y)`` and ``before(r)`` (or ``None``) in one operator, but for the norms that it would pass by, which are called."""
    cols = y.shape[-1]
    pair = lambda norm: (norm.weight, norm.bias)
    inside, eps = {}, 1e-5
    if _fuses(after, cols):
        inside["after"], eps = pair(after), after.eps
    else:
        y = _layer_norm(after, y)
    if before is not None and _fuses(before, cols) and ("after" not in inside or before.eps == eps):
        inside["before"], eps = pair(before), before.eps
    r, n = residual_norm(y, x, scale=scale, eps=eps, **inside)
    return r, n if before is None or "before" in inside else _layer_norm(before, r)
