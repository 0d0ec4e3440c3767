"""The selective state space block: the short causal convolution in front of it, the selective scan, and the norms around a block
with its gate, scale and residual addition.  No counterpart in the reference; names, ``[N,H,L,*]`` views and in/out states are those
of :func:`fast_weight_sum`, whose recurrence the scan extends by a decay.

Rows (``X``, ``Q``, ``K``, ``V``, ``delta``, ``Z``, ``y``, ``x``, ``gate``) are fp32, fp16 or bf16, all of a call alike; parameters, the scan's state and every sum
are fp32.  Views are read in place as long as their last axis is contiguous, and results take the memory order of the rows they belong to (steps outermost
for the permuted views that a layer hands over).  ``lengths`` (int64 ``[N]``, on the GPU, values beyond ``0 .. L`` are cut to it) marks a padded batch: the rows of sequence ``n``
from ``lengths[n]`` on are not read, whatever they hold, their results and gradients are zero, and its states are those after its last row.
States are updated in place and get no gradient; gradients cannot be differentiated again, and tensors with a tangent
(forward-mode differentiation) are refused.  Anything else raises ``FwpError``.
"""
from . import _lib
from .fast_weight import _fwp_torch

_ACTIVATIONS = {None: 0, "sigmoid": 1, "silu": 2}


def _native():
    if _fwp_torch is None:
        raise _lib.FwpError("recurrent-fwp_amd/_fwp_torch.so is missing: build it with recurrent-fwp_amd/csrc/build_torch.sh "
                            "(there is no CPU or PyTorch fallback for these operators)")
    return _fwp_torch


def causal_conv(X, weight, bias=None, state=None, silu=False, lengths=None):
    """``Y[t] = act(bias + sum_j weight[j] X[t - K + 1 + j])`` for every channel, ``act`` the identity or ``x sigmoid(x)``.

    X ``[N,H,L,D]``; weight ``[H,D,K]`` with 1 to 8 taps (the last one meets the newest row); bias ``[H,D]``.  ``state [N,H,K-1,D]``, contiguous and of X's
    type, holds the rows before the first on entry and the last K-1 rows on return (``None``: zeros, not kept): a prompt and single tokens (L = 1)
    continue one another.  Gradients flow to X, weight and bias."""
    return _native().causal_conv(X, weight, bias, state, silu, lengths)


def selective_scan(Q, K, V, delta, A, W=None, D=None, Z=None, delta_bias=None, softplus=False, lengths=None):
    """Per step ``W = exp(dt A) W + k (x) (dt v)``, ``out = W^T q + D v`` (times ``Z sigmoid(Z)``), ``dt = delta + delta_bias`` or its softplus.

    Q, K ``[N,H,L,E]``, E up to 64; V, delta, Z ``[N,H,L,M]``; A ``[H,E,M]``, the decay of every entry of the state, not positive; D, delta_bias ``[H,M]``.
    ``W [N,H,E,M]`` (contiguous, fp32) is the state on entry and the one after the last step on return (``None``: zeros, not kept).  Heads with
    their own q and k are groups of channels; one group of all channels is H = 1.  Gradients flow to everything but W."""
    return _native().selective_scan(Q, K, V, delta, A, W, D, Z, delta_bias, softplus, lengths)


def _weights(norm):
    """(weight, bias) of a norm given as a weight, as such a pair, or not at all."""
    if not isinstance(norm, (tuple, list)):
        return norm, None
    if len(norm) != 2:
        raise _lib.FwpError("a norm is its weight or the pair (weight, bias)")
    return norm


def residual_norm(y, x, after=None, gate=None, scale=None, before=None, eps=1e-5, rms=False, activation=None):
    """``r = x + scale act(gate) norm_after(y)`` and ``n = norm_before(r)``: what lies between the output ``y`` of a block and the input
    ``n`` of the next one on the residual stream ``x``.  Returns ``(r, n)``, or ``(r, None)`` without ``before``.

    y, x ``[..., cols]``, cols up to 8192; x may be fp32 beside narrower rows, and r has its type.  ``after`` and ``before``: a weight ``[cols]`` or a pair
    (weight, bias), ``None``: no norm there.  The norms are LayerNorms, with ``rms`` divisions by the root mean square.  gate ``[..., cols]`` or
    ``[..., 1]`` through ``activation`` (``None``, ``"sigmoid"``, ``"silu"``); scale ``[cols]``.  Gradients flow to every tensor."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise _lib.FwpError(f"activation must be None, 'sigmoid' or 'silu', got {activation!r}")
    (aw, ab), (bw, bb) = _weights(after), _weights(before)
    return _native().residual_norm(y, x, gate, scale, aw, ab, bw, bb, eps, rms, act)
