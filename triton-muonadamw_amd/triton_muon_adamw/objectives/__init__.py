"""Objectives of a training step: losses over rows of logits, with their gradients (gfx950 HIP kernels)."""

from .hip_objectives import (
    PolicyLoss,
    PreferenceLoss,
    distill_loss,
    policy_loss,
    preference_loss,
    token_logprobs,
)

__all__ = ["PolicyLoss", "PreferenceLoss", "distill_loss", "policy_loss", "preference_loss", "token_logprobs"]
