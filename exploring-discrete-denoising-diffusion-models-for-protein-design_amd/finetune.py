"""Fine-tuning objectives at a denoiser's (or a language model's) logits, with the loss modules' manner of the
package: the gradient at the logits comes out of the launch that computes the loss.

  token_logprobs    log-probabilities of given tokens (the reference and old models' side of the losses below)
  TopKDistillLoss   distillation from a teacher's top logits
  PreferenceLoss    pairs of sequences, the first of each preferred: -log sigmoid of the difference of log-ratios
  PolicyLoss        clipped ratio of new to old probabilities times an advantage, with a KL term

Logits are float32, float16 or bfloat16 ``[..., V]`` on the GPU with any strides (where the classes do not lie side by
side, or the positions of a sequence do not follow each other with one stride, they are copied into rows once, and the
copy is kept for the gradient in their place); everything is computed in float32 (the join of a row's lanes, sums over rows
and over sequences in float64) and the gradient is rounded once, to the logits' type.  ``mask`` (bool, the tokens' shape)
says which positions count: the others' logits and labels are not looked at (they may hold NaN, or tokens that are none),
their outputs and gradients are 0, whatever their upstream gradient.  Tokens and classes outside ``[0, V)`` are clamped into it
(a negative ``teacher_index`` marks an entry that is not there).  Only the logits are differentiated, in reverse mode and
once: any other floating input that requires a gradient, a forward-mode tangent and the gradient of a gradient are
refused.

``out_scale=`` multiplies a loss and its gradient.  The gradient of the launch is that for an upstream gradient of 1,
so a constant factor (a loss scaler's, 1 / accumulated batches) costs nothing there, while any other upstream gradient
makes ``backward`` compute the gradient again."""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from ._ops import ops


def _temperature(x: float) -> float:
    x = float(x)
    if not 1e-6 <= x <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6], got {x}")
    return x


def _keep(module: torch.nn.Module, **values) -> None:
    """Plain attributes of a module.  They are no parameters, and ``Module.__setattr__``'s search for them is a third of
    the host time of a forward call."""
    module.__dict__.update(values)


def _finite(x: float, what: str) -> float:
    x = float(x)
    if not math.isfinite(x):
        raise ValueError(f"{what} must be finite, got {x}")
    return x


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, mask: Optional[torch.Tensor] = None,
                   temperature: float = 1.0) -> torch.Tensor:
    """``log_softmax(logits / temperature)`` at ``tokens`` (logits ``[..., V]``, tokens ``[...]``), float32 of the
    tokens' shape, 0 where ``mask`` is false; differentiable by the logits."""
    _lib.require_device(logits, tokens, mask)
    return ops.token_logprobs(logits, tokens, mask, _temperature(temperature))


class TopKDistillLoss(torch.nn.Module):
    """Distillation from the ``k`` best logits that a teacher gave per position.

    With ``q = softmax(teacher_logits / temperature)`` over the kept entries of a position (those with an index of at
    least 0 and a logit above -inf), ``forward`` returns the mean over the counted positions of
    ``temperature**2 * KL(q || softmax(logits / temperature))``, times ``out_scale``.  logits ``[..., V]``,
    teacher_logits and teacher_index ``[..., k]`` with k up to 256; a class listed twice has the sum of its entries,
    a position that keeps none adds 0.  ``per_token`` holds the positions' terms of the last call."""

    def __init__(self, temperature: float = 1.0):
        super().__init__()
        _keep(self, temperature=_temperature(temperature), per_token=None)

    def forward(self, logits, teacher_logits, teacher_index, mask=None, out_scale=1.0):
        _lib.require_device(logits, teacher_logits, teacher_index, mask)
        loss, per_token = ops.topk_distill_loss(logits, teacher_logits, teacher_index, mask, self.temperature,
                                                _finite(out_scale, "out_scale"))
        _keep(self, per_token=per_token)
        return loss


class PolicyLoss(torch.nn.Module):
    """Clipped policy loss with a KL term.

    With ``lp`` the tokens' log-probabilities at ``temperature``, ``r = exp(lp - old_logprobs)`` and
    ``x = ref_logprobs - lp``, ``forward`` returns the mean over the counted positions of
    ``-min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A) + kl_coeff * (exp(x) - x - 1)``, times ``out_scale``.
    logits ``[..., V]``; tokens, old_logprobs, ref_logprobs ``[...]``; advantages ``[...]``, or ``[B]`` for one per
    sequence of tokens ``[B, L]``.  ``logprobs`` holds ``lp`` of the last call (0 where a position is not counted)."""

    def __init__(self, clip_low: float = 0.2, clip_high: float = 0.2, kl_coeff: float = 0.0, temperature: float = 1.0):
        super().__init__()
        clip_low, clip_high = _finite(clip_low, "clip_low"), float(clip_high)
        if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
            raise ValueError(f"clip range [1 - {clip_low}, 1 + {clip_high}]: need 0 <= clip_low <= 1, clip_high >= 0")
        _keep(self, clip_low=clip_low, clip_high=clip_high, kl_coeff=_finite(kl_coeff, "kl_coeff"),
              temperature=_temperature(temperature), logprobs=None)

    def forward(self, logits, tokens, old_logprobs, advantages, ref_logprobs=None, mask=None, out_scale=1.0):
        _lib.require_device(logits, tokens, old_logprobs, advantages, ref_logprobs, mask)
        if self.kl_coeff != 0.0 and ref_logprobs is None:
            raise ValueError("kl_coeff needs ref_logprobs")
        loss, logprobs = ops.policy_loss(logits, tokens, old_logprobs, advantages, ref_logprobs, mask, self.temperature,
                                         self.clip_low, self.clip_high, self.kl_coeff, _finite(out_scale, "out_scale"))
        _keep(self, logprobs=logprobs)
        return loss


class PreferenceLoss(torch.nn.Module):
    """Preference loss of pairs of sequences.

    logits ``[2 P, L, V]`` and tokens ``[2 P, L]`` hold the P preferred sequences first, then in the same order the
    ones that they are preferred to; ref_logprobs ``[2 P, L]`` are the tokens' log-probabilities under the reference
    model (``token_logprobs``; None: 0).  With ``D`` a sequence's sum of ``lp - ref_logprobs`` over its counted
    positions (their mean with ``average``) and ``m = beta * (D_preferred - D_other)``, ``forward`` returns the mean
    over the pairs of ``-(1 - label_smoothing) * log sigmoid(m) - label_smoothing * log sigmoid(-m)``, times
    ``out_scale`` (a term of weight 0 is left out, also where its logarithm is infinite).  ``rewards`` holds ``beta * D`` ``[2 P]`` of the last call."""

    def __init__(self, beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False):
        super().__init__()
        beta, label_smoothing = _finite(beta, "beta"), _finite(label_smoothing, "label_smoothing")
        if not 0.0 <= label_smoothing <= 1.0:
            raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
        _keep(self, beta=beta, label_smoothing=label_smoothing, average=bool(average), rewards=None)

    def forward(self, logits, tokens, ref_logprobs=None, mask=None, out_scale=1.0):
        _lib.require_device(logits, tokens, ref_logprobs, mask)
        loss, rewards = ops.preference_loss(logits, tokens, ref_logprobs, mask, self.beta, self.label_smoothing,
                                            self.average, _finite(out_scale, "out_scale"))
        _keep(self, rewards=rewards)
        return loss
