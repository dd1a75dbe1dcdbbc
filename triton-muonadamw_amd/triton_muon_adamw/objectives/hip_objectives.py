"""Losses over rows of logits: the part of a training step before the optimizer.

The reference starts at gradients; these have no counterpart there.  Logits
are ``(rows, vocab)`` or ``(batch, length, vocab)`` in float32, bfloat16 or
float16, with any strides but a contiguous vocabulary; what goes with them has
one value for each row, may be broadcast and is taken as a constant.  Between the logits and the
gradient, which has the logits' type, everything is float32.  Work is queued on
the current stream without a host synchronisation, results do not depend on
the order in which anything runs, and a HIP graph can record a pass.

Rows whose token is ``ignore_index`` (or whose mask is false) are not read:
infinities and NaN in them change nothing, and where no row is left the loss is
0.  Values on the device are not looked at by the host, so a token beyond the
vocabulary cannot raise: it reads nothing and gives NaN.
"""

from __future__ import annotations

from typing import Literal, NamedTuple

import torch

from .. import _lib

_KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}


class PolicyLoss(NamedTuple):
    """``loss`` carries the gradient; the rest are values for the log."""

    loss: torch.Tensor
    logprobs: torch.Tensor  # of the tokens, 0 where they do not count
    kl: torch.Tensor        # mean of exp(ref - logprob) - (ref - logprob) - 1, 0 without ref_logprobs
    clipped: torch.Tensor   # share of the tokens that the clamp keeps from contributing


class PreferenceLoss(NamedTuple):
    """``loss`` carries the gradient; the rest are values for the log, one a sequence."""

    loss: torch.Tensor
    logprobs: torch.Tensor  # sums (or means) over each sequence's tokens
    rewards: torch.Tensor   # beta * (logprobs - ref_logprobs)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                   entropy: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Log-probability of ``tokens`` under ``softmax(logits / temperature)``,
    float32, 0 where the token is ``ignore_index``; with ``entropy`` also the
    distribution's entropy.  Both are differentiable; rows whose gradients from
    outside are 0 get one of 0, whatever their logits."""
    out = _lib.objectives().token_logprobs(logits, tokens, temperature, ignore_index, entropy)
    return out if entropy else out[0]


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: torch.Tensor | None = None, kl_coef: float = 0.0,
                clip: tuple[float, float] = (0.2, 0.2), average: Literal["token", "sequence"] = "token",
                offsets: torch.Tensor | None = None, temperature: float = 1.0, ignore_index: int = -100,
                scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss: with ``ratio = exp(logprob - old_logprobs)``, the mean of
    ``-min(ratio * A, clamp(ratio, 1 - clip[0], 1 + clip[1]) * A)`` plus, with
    ``ref_logprobs``, ``kl_coef * (exp(d) - d - 1)`` for ``d = ref_logprobs - logprob``.

    The mean is over all tokens that count, or with ``average="sequence"`` over
    the sequences' own means (those with a token that counts): one for each
    element of the batch, or for ``(rows, vocab)`` logits from ``offsets[i]`` to
    ``offsets[i + 1]``.  ``scale`` multiplies the loss; a factor that is known
    beforehand (of gradient accumulation, for one) is given here rather than
    multiplied afterwards, which has the gradient computed a second time."""
    if average not in ("token", "sequence"):
        raise ValueError(f"average must be 'token' or 'sequence' (got {average!r})")
    return PolicyLoss(*_lib.objectives().policy_loss(
        logits, tokens, old_logprobs, advantages, ref_logprobs, kl_coef, clip[0], clip[1], average == "sequence",
        offsets, temperature, ignore_index, scale))


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, ref_logprobs: torch.Tensor | None, *,
                    beta: float = 0.1, kind: Literal["sigmoid", "ipo", "hinge"] = "sigmoid",
                    label_smoothing: float = 0.0, length_average: bool = False, offsets: torch.Tensor | None = None,
                    temperature: float = 1.0, ignore_index: int = -100) -> PreferenceLoss:
    """Preference loss over pairs: of ``2 P`` sequences the first ``P`` are the
    preferred ones, sequence ``i`` against ``i + P``.  A sequence's reward is
    ``beta * (logprob - ref_logprobs)`` with the sum (``length_average``: the
    mean) of its tokens' log-probabilities; ``h`` is the difference of a pair's.

    ``kind``: ``"sigmoid"`` ``-log sigmoid(h)`` (with ``label_smoothing`` e,
    ``1 - e`` of it and ``e`` of ``-log sigmoid(-h)``), ``"ipo"``
    ``(h / beta - 1 / (2 beta))**2``, ``"hinge"`` ``max(0, 1 - h)``; the loss is
    the mean over the pairs.  Sequences as in :func:`policy_loss`; rows in none of
    them do not count.  ``ref_logprobs`` holds one value for each, ``None`` for 0."""
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)} (got {kind!r})")
    return PreferenceLoss(*_lib.objectives().preference_loss(
        logits, tokens, ref_logprobs, beta, _KINDS[kind], label_smoothing, length_average, offsets, temperature,
        ignore_index))


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor, *,
                 teacher_lse: torch.Tensor | None = None, mask: torch.Tensor | None = None, temperature: float = 1.0,
                 scale: float = 1.0) -> torch.Tensor:
    """``temperature**2`` times the mean divergence KL(teacher || student) at
    ``temperature``, from the teacher's ``k`` first logits of each row and their
    places in the vocabulary (``k`` up to 1024, in any order).

    Without ``teacher_lse`` the ``k`` entries are the teacher's whole distribution.
    With ``teacher_lse``, the ``logsumexp(teacher / temperature)`` over its whole
    vocabulary, they have their true probabilities, and all other entries
    together count as one more, of which at least ``2**-20`` is taken to be left.
    Entries with a negative index or a logit of ``-inf`` are padding.  Rows with a
    false ``mask`` do not count.  ``scale`` as in :func:`policy_loss`."""
    return _lib.objectives().distill_loss(logits, teacher_logits, teacher_indices, teacher_lse, mask, temperature,
                                          scale)[0]
