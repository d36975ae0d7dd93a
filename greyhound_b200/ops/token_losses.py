"""Clipped policy loss and preference loss: custom ops + autograd Functions.

The forward computes the loss and, for the policy loss, the unweighted
gradient of every token; the backward applies the reduction's weight and the
incoming gradient in one pass.
"""

from __future__ import annotations

from typing import Any

import torch
from torch import Tensor

from greyhound_b200.kernels.token_losses import (
    policy_loss_backward,
    policy_loss_forward,
    policy_workspace_bytes,
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
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(loss, stats [4], unweighted token gradients (empty if not wanted), workspace)."""
    loss, stats, d, ws = policy_loss_forward(
        logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, clip_low, clip_high, kl_multiplier,
        reduction, advantages_per, want_grad,
    )
    return loss, stats, stats.new_empty(0) if d is None else d, ws


@clipped_policy_loss_fwd.register_fake
def _(logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, clip_low, clip_high, kl_multiplier,
      reduction, advantages_per, want_grad):
    dev = logprobs.device
    return (
        _scalar(logprobs),
        torch.empty([4], dtype=torch.float32, device=dev),
        torch.empty([logprobs.numel() if want_grad else 0], dtype=torch.float32, device=dev),
        torch.empty(policy_workspace_bytes(logprobs, cu_seqlens, reduction), dtype=torch.uint8, device=dev),
    )


@torch.library.custom_op("greyhound::clipped_policy_loss_bwd", mutates_args=())
def clipped_policy_loss_bwd(
    dlogprobs: Tensor,
    stats: Tensor,
    workspace: Tensor,
    cu_seqlens: Tensor | None,
    grad_output: Tensor,
    shape: list[int],
    dtype: torch.dtype,
    reduction: str,
) -> Tensor:
    return policy_loss_backward(dlogprobs, stats, workspace, cu_seqlens, grad_output, shape, dtype, reduction)


@clipped_policy_loss_bwd.register_fake
def _(dlogprobs, stats, workspace, cu_seqlens, grad_output, shape, dtype, reduction):
    return torch.empty(shape, dtype=dtype, device=dlogprobs.device)


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
        clip_low: float,
        clip_high: float,
        kl_multiplier: float,
        reduction: str,
        advantages_per: str,
    ) -> tuple[Tensor, Tensor]:
        loss, stats, d, ws = clipped_policy_loss_fwd(
            logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens, clip_low, clip_high, kl_multiplier,
            reduction, advantages_per, ctx.needs_input_grad[0],
        )
        if ctx.needs_input_grad[0]:
            cu = None if cu_seqlens is None else cu_seqlens.contiguous()
            ctx.save_for_backward(d, stats, ws, cu)
            ctx.shape, ctx.dtype, ctx.reduction = list(logprobs.shape), logprobs.dtype, reduction
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: Tensor, _: Tensor):  # type: ignore[override]
        d, stats, ws, cu = ctx.saved_tensors
        grad = clipped_policy_loss_bwd(d, stats, ws, cu, grad_output, ctx.shape, ctx.dtype, ctx.reduction)
        return grad, None, None, None, None, None, None, None, None, None, None


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
) -> tuple[Tensor, Tensor, Tensor]:
    """(loss, rewards [sequences], gradient of a valid token [sequences])."""
    return preference_loss_forward(
        logprobs, ref_logprobs, mask, cu_seqlens, beta, loss_type, label_smoothing, margin, length_normalized,
        reduction,
    )


@preference_loss_fwd.register_fake
def _(logprobs, ref_logprobs, mask, cu_seqlens, beta, loss_type, label_smoothing, margin, length_normalized,
      reduction):
    seqs = cu_seqlens.shape[0] - 1 if cu_seqlens is not None else logprobs.shape[0]
    per = [torch.empty([seqs], dtype=torch.float32, device=logprobs.device) for _ in range(2)]
    return _scalar(logprobs), per[0], per[1]


@torch.library.custom_op("greyhound::preference_loss_bwd", mutates_args=())
def preference_loss_bwd(
    coef: Tensor,
    grad_output: Tensor,
    mask: Tensor | None,
    cu_seqlens: Tensor | None,
    shape: list[int],
    dtype: torch.dtype,
) -> Tensor:
    return preference_loss_backward(coef, grad_output, mask, cu_seqlens, shape, dtype)


@preference_loss_bwd.register_fake
def _(coef, grad_output, mask, cu_seqlens, shape, dtype):
    return torch.empty(shape, dtype=dtype, device=coef.device)


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
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
        loss, rewards, coef = preference_loss_fwd(
            logprobs, ref_logprobs, mask, cu_seqlens, beta, loss_type, label_smoothing, margin, length_normalized,
            reduction,
        )
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(coef, mask, cu_seqlens)
            ctx.shape, ctx.dtype = list(logprobs.shape), logprobs.dtype
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_output: Tensor, _: Tensor):  # type: ignore[override]
        coef, mask, cu = ctx.saved_tensors
        grad = preference_loss_bwd(coef, grad_output, mask, cu, ctx.shape, ctx.dtype)
        return grad, None, None, None, None, None, None, None, None, None
