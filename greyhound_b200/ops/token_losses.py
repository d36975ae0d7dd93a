"""Clipped policy loss and preference loss: custom ops + autograd Functions.

The forward computes the loss and, for the policy loss, the unweighted
gradient of every token; the backward applies the reduction's weight and the
incoming gradient in one pass.
"""

from __future__ import annotations

from typing import Any

import torch
from torch import Tensor

from greyhound_b200 import _lib
from greyhound_b200.kernels.token_losses import (
    policy_loss_backward,
    policy_loss_forward,
    policy_state_size,
    preference_loss_backward,
    preference_loss_forward,
)

__all__ = [
    "ClippedPolicyLossFunction",
    "PreferenceLossFunction",
    "clipped_policy_loss_bwd",
    "clipped_policy_loss_fwd",
    "preference_loss_bwd",
    "preference_loss_fwd",
]


def _scalar(t: Tensor) -> Tensor:
    return torch.empty([], dtype=torch.float32, device=t.device)


@torch.library.custom_op("greyhound::clipped_policy_loss_fwd", mutates_args=())
def clipped_policy_loss_fwd(
    logprobs: Tensor,
    old_logprobs: Tensor | None,
    advantages: Tensor,
    ref_logprobs: Tensor | None,
    mask: Tensor | None,
    cu_seqlens: Tensor | None,
    clip_low: float,
    clip_high: float,
    kl_multiplier: float,
    reduction: str,
    advantages_per: str,
    want_grad: bool,
) -> tuple[Tensor, Tensor]:
    """(loss, state: mean KL, clipped share, valid tokens, and what the backward reads)."""
    return policy_loss_forward(
        logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, clip_low, clip_high, kl_multiplier,
        reduction, advantages_per, want_grad,
    )


@clipped_policy_loss_fwd.register_fake
def _(logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, clip_low, clip_high, kl_multiplier,
      reduction, advantages_per, want_grad):
    size = policy_state_size(logprobs, cu_seqlens, reduction, want_grad)
    return _scalar(logprobs), torch.empty([size], dtype=torch.float32, device=logprobs.device)


@torch.library.custom_op("greyhound::clipped_policy_loss_bwd", mutates_args=())
def clipped_policy_loss_bwd(
    state: Tensor,
    cu_seqlens: Tensor | None,
    grad_output: Tensor,
    shape: list[int],
    dtype: torch.dtype,
    reduction: str,
) -> Tensor:
    return policy_loss_backward(state, cu_seqlens, grad_output, shape, dtype, reduction)


@clipped_policy_loss_bwd.register_fake
def _(state, cu_seqlens, grad_output, shape, dtype, reduction):
    return torch.empty(shape, dtype=dtype, device=state.device)


class ClippedPolicyLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        logprobs: Tensor,
        old_logprobs: Tensor | None,
        advantages: Tensor,
        ref_logprobs: Tensor | None,
        mask: Tensor | None,
        cu_seqlens: Tensor | None,
        options: tuple[float, float, float, str, str],  # the ops' arguments from clip_low to advantages_per
        grad_enabled: bool = True,  # the caller's mode: in here gradients are always off
    ) -> tuple[Tensor, Tensor]:
        want = grad_enabled and ctx.needs_input_grad[0]
        fwd = policy_loss_forward if _lib.eager(logprobs) else clipped_policy_loss_fwd
        loss, state = fwd(logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, *options, want)
        if want:
            ctx.save_for_backward(state, None if cu_seqlens is None else cu_seqlens.contiguous())
            ctx.like = list(logprobs.shape), logprobs.dtype, options[3]
        ctx.mark_non_differentiable(state)
        ctx.set_materialize_grads(False)  # no zeros for state's gradient, which nobody reads
        return loss, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: Tensor, _: Tensor):  # type: ignore[override]
        if grad_output is None:
            return (None,) * 8
        state, cu = ctx.saved_tensors
        bwd = policy_loss_backward if _lib.eager(state) else clipped_policy_loss_bwd
        return bwd(state, cu, grad_output, *ctx.like), None, None, None, None, None, None, None


@torch.library.custom_op("greyhound::preference_loss_fwd", mutates_args=())
def preference_loss_fwd(
    logprobs: Tensor,
    ref_logprobs: Tensor | None,
    mask: Tensor | None,
    cu_seqlens: Tensor | None,
    beta: float,
    loss_type: str,
    label_smoothing: float,
    margin: float,
    length_normalized: bool,
    reduction: str,
) -> tuple[Tensor, Tensor]:
    """(loss, state [2, sequences]: rewards, gradient of a valid token of each sequence)."""
    return preference_loss_forward(
        logprobs, ref_logprobs, mask, cu_seqlens, beta, loss_type, label_smoothing, margin, length_normalized,
        reduction,
    )


@preference_loss_fwd.register_fake
def _(logprobs, ref_logprobs, mask, cu_seqlens, beta, loss_type, label_smoothing, margin, length_normalized,
      reduction):
    seqs = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else logprobs.shape[0]
    return _scalar(logprobs), torch.empty([2, seqs], dtype=torch.float32, device=logprobs.device)


@torch.library.custom_op("greyhound::preference_loss_bwd", mutates_args=())
def preference_loss_bwd(
    state: Tensor,
    grad_output: Tensor,
    mask: Tensor | None,
    cu_seqlens: Tensor | None,
    shape: list[int],
    dtype: torch.dtype,
) -> Tensor:
    return preference_loss_backward(state, grad_output, mask, cu_seqlens, shape, dtype)


@preference_loss_bwd.register_fake
def _(state, grad_output, mask, cu_seqlens, shape, dtype):
    return torch.empty(shape, dtype=dtype, device=state.device)


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        logprobs: Tensor,
        ref_logprobs: Tensor | None,
        mask: Tensor | None,
        cu_seqlens: Tensor | None,
        options: tuple[float, str, float, float, bool, str],  # the ops' arguments from beta on
    ) -> tuple[Tensor, Tensor]:
        fwd = preference_loss_forward if _lib.eager(logprobs) else preference_loss_fwd
        loss, state = fwd(logprobs, ref_logprobs, mask, cu_seqlens, *options)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(state, mask, cu_seqlens)
            ctx.like = list(logprobs.shape), logprobs.dtype
        ctx.mark_non_differentiable(state)
        ctx.set_materialize_grads(False)  # no zeros for state's gradient, which nobody reads
        return loss, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: Tensor, _: Tensor):  # type: ignore[override]
        if grad_output is None:
            return (None,) * 5
        state, mask, cu = ctx.saved_tensors
        bwd = preference_loss_backward if _lib.eager(state) else preference_loss_bwd
        return bwd(state, grad_output, mask, cu, *ctx.like), None, None, None, None
