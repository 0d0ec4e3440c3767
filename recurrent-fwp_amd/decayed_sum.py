"""The block of a decayed sum rule: rotary positions of its queries and keys, the sum rule with a decay for each head, and the norm of every head's channels with
its gate.  No counterpart in the reference; names, ``[N,H,L,*]`` views and in/out states are those of :func:`fast_weight_sum`, which is the rule without
its decay.

Rows (``Q``, ``K``, ``V``, ``X``, ``gate``) are fp32, fp16 or bf16, all of a call alike; decays, parameters, the state and every sum are fp32.  Views are read in place as
long as their last axis is contiguous, and results take the memory order of the rows they belong to (steps outermost for the permuted views that a layer hands
over).  ``lengths`` (int64 ``[N]``, on the GPU, values beyond ``0 .. L`` are cut to it) marks a padded batch: the rows of sequence ``n`` from ``lengths[n]`` on
are not read, whatever they hold, their results and gradients are zero, and its state is the one after its last row.  States are updated in place
and get no gradient; gradients cannot be differentiated again, and tensors with a tangent (forward-mode differentiation) are refused.  Anything else
raises ``FwpError``.
"""
import math

import torch

from . import _lib
from .selective_scan import _ACTIVATIONS, _native


def decayed_sum(Q, K, V, log_decay, W=None, scale=1.0, lengths=None):
    """Per step and head ``W = exp(log_decay) W + k (x) v``, ``out = scale W^T q``.

    Q, K ``[N,.,L,E]``, E up to 128; V ``[N,.,L,M]``; ``log_decay [H]``, one decay for each head, or ``[N,H,L]``, one for each step of a head: fp32, not positive, and minus infinity
    empties the state.  Q, K and V have H heads each or a part of them: with G of them, head ``h`` takes head ``h // (H // G)``.  ``W [N,H,E,M]`` (contiguous, fp32) is the
    state on entry and the one after the last step on return (``None``: zeros, not kept): a prompt and single tokens (L = 1) continue one another.  Returns ``[N,H,L,M]``;
    gradients flow to Q, K, V and log_decay.

    A number that is not finite makes infinite or NaN what depends on it, and leaves the results of the steps before it as they are; gradients are NaN in its whole chunk,
    up to 63 steps before and behind it.  fp32 numbers beyond 3.39e38 may count as infinite where there are more than 32 keys."""
    return _native().decayed_sum(Q, K, V, log_decay, W, scale, lengths)


def rotary(Q, K, frequencies, positions=None, interleaved=False, scale=1.0, lengths=None):
    """Turns the first ``2 * len(frequencies)`` channels of every row, pair by pair, by ``position * frequencies`` radians, and multiplies them by ``scale``; the other
    channels stay.  Returns ``(q, k)``, or ``(q, None)`` where K is ``None``.

    Q, K ``[N,.,L,D]``; frequencies fp64 (:func:`rotary_frequencies`); a pair is channels ``i`` and ``i + len(frequencies)``, or ``2i`` and ``2i + 1`` if ``interleaved``.
    Step t of sequence n is at position t, at ``positions[n] + t`` with positions ``[N]``, at ``positions[n, t]`` with positions ``[N,L]`` (int64).  Gradients flow to Q
    and K."""
    return _native().rotary(Q, K, frequencies, positions, interleaved, scale, lengths)


def rotary_frequencies(width, base=10000.0, scaling=None, factor=1.0, trained=None, turns=(1.0, 32.0), device=None):
    """``(frequencies, scale)`` for :func:`rotary` to turn ``width`` channels: pair i turns by ``base ** (-2 i / width)`` radians a position, and ``scale`` is what the
    turned channels are multiplied by.  For contexts ``factor`` times as long as those of training:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: ``base`` times ``factor ** (width / (width - 2))``, which slows the slowest pair by ``factor`` and leaves the fastest;
    * ``"parts"``: pairs that turn more than ``turns[1]`` times over the ``trained`` positions stay, those that turn less than ``turns[0]`` times are slowed by ``factor``, those
      between by a linear share of it, and ``scale`` is ``1 + 0.1 ln(factor)``."""
    if width < 2 or width % 2:
        raise _lib.FwpError(f"an even number of channels turns, got {width}")
    if scaling not in (None, "linear", "base", "parts"):
        raise _lib.FwpError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
    if not factor > 0 or not base > 0:
        raise _lib.FwpError("base and factor must be positive")
    scale = 1.0
    if scaling == "base":
        base = base * factor ** (width / max(width - 2, 1))
    f = base ** (-2.0 * torch.arange(width // 2, dtype=torch.float64, device=device) / width)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if trained is None or not turns[1] > turns[0]:
            raise _lib.FwpError("scaling by parts needs the trained length, and turns in ascending order")
        kept = ((trained * f / (2 * math.pi) - turns[0]) / (turns[1] - turns[0])).clamp(0, 1)
        f, scale = f * (kept + (1 - kept) / factor), 1 + 0.1 * math.log(factor)
    return f, scale


def group_norm(X, groups, weight=None, bias=None, gate=None, eps=1e-5, rms=False, activation=None):
    """Every row's channels in ``groups`` groups, each normalised by its own mean and variance (``rms``: divided by its root mean square), times ``weight`` plus ``bias``; then
    times ``act(gate)``, or ``act`` of it where there is no gate.

    X, gate ``[..., channels]``, channels last; a row is normalised by itself, so that no step sees another.  weight, bias ``[channels]``; groups of up to 1024 channels, at most 2^30 rows.
    ``activation``: ``None``, ``"sigmoid"`` or ``"silu"``.  Gradients flow to every tensor."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise _lib.FwpError(f"activation must be None, 'sigmoid' or 'silu', got {activation!r}")
    return _native().group_norm(X, groups, weight, bias, gate, eps, rms, act)
