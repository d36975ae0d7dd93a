"""Public functional API — same signatures and semantics as src/greyhound/nn/functional.py.

``selective_log_softmax`` (:53-69), ``cross_entropy`` (:72-116),
``autograd_loss_and_logits_grad`` (:119-148), ``chunked_linear_loss`` (:151-223)
and ``chunked_linear_cross_entropy`` (:226-287).
``chunked_linear_selective_log_softmax``, ``clipped_policy_loss`` and
``preference_loss`` have no counterpart there. ``weight`` is ``[V, D]`` and is
handed to the ops as the ``[D, V]`` view ``weight.T``, exactly as the reference
does, so the op schemas and their fakes are unchanged.
"""

from __future__ import annotations

from collections.abc import Callable
from typing import Any, Literal, NamedTuple, cast

import torch
from torch import Tensor

from greyhound_b200.kernels.token_losses import _no_grad_to
from greyhound_b200.ops.chunked_linear_cross_entropy import ChunkedLinearCrossEntropyFunction
from greyhound_b200.ops.chunked_linear_loss import ChunkedLinearLossFunction
from greyhound_b200.ops.chunked_linear_selective_log_softmax import ChunkedLinearSelectiveLogSoftmaxFunction
from greyhound_b200.ops.cross_entropy import CrossEntropyFunction
from greyhound_b200.ops.logprobs import SelectiveLogSoftmaxFunction
from greyhound_b200.ops.token_losses import ClippedPolicyLossFunction, PreferenceLossFunction

__all__ = [
    "selective_log_softmax",
    "cross_entropy",
    "autograd_loss_and_logits_grad",
    "chunked_linear_loss",
    "chunked_linear_cross_entropy",
    "chunked_linear_selective_log_softmax",
    "clipped_policy_loss",
    "preference_loss",
    "PolicyLossMetrics",
    "PreferenceRewards",
]


class PolicyLossMetrics(NamedTuple):
    """0-d fp32 tensors over the valid tokens, without gradients."""

    kl: Tensor  # mean of e^u - u - 1, u = ref - logprob (0 without ref_logprobs)
    clip_fraction: Tensor  # share of tokens whose ratio is clipped
    tokens: Tensor  # their number


class PreferenceRewards(NamedTuple):
    """``[pairs]`` fp32 tensors, without gradients: beta times each sequence's log ratio."""

    chosen: Tensor
    rejected: Tensor


def _slice_chunk_arg(value: Any, start: int, end: int, batch_size: int) -> Any:
    if isinstance(value, Tensor) and value.ndim > 0 and value.shape[0] == batch_size:
        return value[start:end]
    return value


def _check_scalar_loss(loss: Tensor) -> None:
    if loss.ndim != 0:
        raise ValueError(f"chunked loss function must return a scalar tensor, got {loss.shape}")


def _check_accum_dtype(grad_weight_accum_dtype: str) -> None:
    if grad_weight_accum_dtype not in ("fp32", "weight"):
        raise ValueError(
            "grad_weight_accum_dtype must be either 'fp32' or 'weight', "
            f"got {grad_weight_accum_dtype!r}"
        )


def selective_log_softmax(logits: Tensor, index: Tensor) -> Tensor:
    """Log-probability of ``index`` under ``softmax(logits)`` along the last dim.

    Equivalent to ``gather(logits.log_softmax(-1), -1, index[..., None])[..., 0]``
    without materialising the log-probabilities: one streaming fp32
    log-sum-exp per row. Output has ``index``'s shape and the logits dtype.
    Differentiable with respect to ``logits``.
    """
    return cast(Tensor, SelectiveLogSoftmaxFunction.apply(logits, index))


def cross_entropy(
    logits: Tensor,
    target: Tensor,
    ignore_index: int = -100,
    reduction: Literal["sum", "mean"] = "mean",
    z_loss_multiplier: float = 0.0,
) -> Tensor:
    """Cross-entropy of materialised ``[B, V]`` logits, plus optional z-loss.

    ``loss = sum_valid(lse - logits[target]) + z_loss_multiplier * sum_valid(lse^2)``,
    divided by the number of valid (``target != ignore_index``) rows when
    ``reduction="mean"``. The logits gradient is produced in the same pass and
    returned by autograd; the input ``logits`` tensor is never modified.
    """
    return cast(
        Tensor,
        CrossEntropyFunction.apply(logits, target, ignore_index, reduction, z_loss_multiplier),
    )


def autograd_loss_and_logits_grad(
    loss_fn: Callable[..., Tensor],
) -> Callable[..., tuple[Tensor, Tensor]]:
    """Wrap a scalar loss ``loss_fn(logits, *args, **kwargs)`` to return ``(loss, dloss/dlogits)``."""

    def loss_and_grad(logits: Tensor, *args: Any, **kwargs: Any) -> tuple[Tensor, Tensor]:
        with torch.enable_grad():
            logits_for_grad = logits.detach().requires_grad_(True)
            loss = loss_fn(logits_for_grad, *args, **kwargs)
            _check_scalar_loss(loss)
            (grad_logits,) = torch.autograd.grad(loss, logits_for_grad)
        return loss.detach(), grad_logits.detach()

    return loss_and_grad


def chunked_linear_loss(
    inputs: Tensor,
    weight: Tensor,
    loss_and_grad_fn: Callable[..., tuple[Tensor, Tensor]],
    *loss_args: Any,
    chunk_size: int | None = None,
    grad_weight_accum_dtype: Literal["fp32", "weight"] = "fp32",
    **loss_kwargs: Any,
) -> Tensor:
    """Row-chunked ``inputs @ weight.T`` followed by a user loss-and-gradient callback.

    For each row chunk the callback gets ``(logits_chunk, *args, **kwargs)``,
    with every tensor argument whose leading dim equals ``inputs.shape[0]``
    sliced to the chunk's rows, and returns ``(scalar_loss, grad_logits)``.
    Input and weight gradients are accumulated chunk by chunk (weight gradient
    in fp32 unless ``grad_weight_accum_dtype="weight"``). Returns the summed loss.
    """
    _check_accum_dtype(grad_weight_accum_dtype)
    batch_size = inputs.shape[0]

    def chunk_loss_and_grad_fn(logits_chunk: Tensor, start: int, end: int) -> tuple[Tensor, Tensor]:
        chunk_args = tuple(_slice_chunk_arg(a, start, end, batch_size) for a in loss_args)
        chunk_kwargs = {k: _slice_chunk_arg(v, start, end, batch_size) for k, v in loss_kwargs.items()}
        return loss_and_grad_fn(logits_chunk, *chunk_args, **chunk_kwargs)

    return cast(
        Tensor,
        ChunkedLinearLossFunction.apply(
            inputs, weight.T, chunk_loss_and_grad_fn, chunk_size, grad_weight_accum_dtype == "fp32"
        ),
    )


def chunked_linear_cross_entropy(
    inputs: Tensor,
    weight: Tensor,
    target: Tensor,
    ignore_index: int = -100,
    reduction: Literal["sum", "mean"] = "mean",
    z_loss_multiplier: float = 0.0,
    grad_weight_accum_dtype: Literal["fp32", "weight"] = "fp32",
) -> Tensor:
    """Cross-entropy of ``inputs @ weight.T`` without keeping the logits.

    ``inputs`` is ``[BT, D]``, ``weight`` is ``[V, D]``, ``target`` is ``[BT]``
    with class ids in ``[0, V)`` or ``ignore_index``. The forward computes the
    loss and, when an input requires grad, both gradients; ``backward`` only
    scales them by the incoming gradient. ``grad_weight_accum_dtype="fp32"``
    accumulates the weight gradient in fp32 and casts once; ``"weight"``
    accumulates in the parameter dtype.
    """
    _check_accum_dtype(grad_weight_accum_dtype)
    return cast(
        Tensor,
        ChunkedLinearCrossEntropyFunction.apply(
            inputs,
            weight.T,
            target,
            ignore_index,
            reduction,
            z_loss_multiplier,
            grad_weight_accum_dtype == "fp32",
        ),
    )


def chunked_linear_selective_log_softmax(
    inputs: Tensor,
    weight: Tensor,
    index: Tensor,
    ignore_index: int = -100,
    temperature: float = 1.0,
    grad_weight_accum_dtype: Literal["fp32", "weight"] = "fp32",
) -> Tensor:
    """Log-probability of ``index`` under ``softmax(inputs @ weight.T / temperature)``.

    ``selective_log_softmax`` from hidden states, without the logits:
    ``inputs`` is ``[..., D]`` and ``weight`` ``[V, D]``, both bf16 or both
    fp16, with ``D`` a multiple of 8; ``index`` has ``inputs``' leading shape,
    int32 or int64. The result has ``index``'s shape and is fp32, computed from
    unrounded fp32 logits (ratios of probabilities need more than 16 bits).

    Positions where ``index == ignore_index`` give 0 and no gradient, whatever
    their hidden state holds. An index outside ``[0, V)`` gives NaN and no
    gradient, and the next call on the device raises ``ValueError``.

    Differentiable (once) with respect to ``inputs`` and ``weight``, for any
    gradient of the log-probabilities. Up to ``N * V * 2`` bytes of 4 GiB the
    forward keeps ``e^x`` for that; otherwise the backward recomputes the logits
    in row chunks. The weight gradient is summed over chunks in fp32 or, with
    ``grad_weight_accum_dtype="weight"``, in the parameter's type.
    """
    _check_accum_dtype(grad_weight_accum_dtype)
    if inputs.ndim < 1 or index.shape != inputs.shape[:-1]:
        raise ValueError(f"expected index shape {tuple(inputs.shape[:-1])}, got {tuple(index.shape)}")
    flat, flat_index = inputs, index
    if inputs.ndim != 2:  # not for two dimensions: a view is a step of autograd's, both ways
        flat = inputs.reshape(index.numel(), inputs.shape[-1])
        flat_index = index.reshape(-1)
    out = cast(
        Tensor,
        ChunkedLinearSelectiveLogSoftmaxFunction.apply(
            flat, weight, flat_index, ignore_index, float(temperature), grad_weight_accum_dtype == "fp32",
            torch.is_grad_enabled(),
        ),
    )
    return out if inputs.ndim == 2 else out.reshape(index.shape)


def clipped_policy_loss(
    logprobs: Tensor,
    old_logprobs: Tensor | None,
    advantages: Tensor,
    ref_logprobs: Tensor | None = None,
    mask: Tensor | None = None,
    cu_seqlens: Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_multiplier: float = 0.0,
    reduction: Literal["sum", "mean", "sequence_mean"] = "mean",
    advantages_per: Literal["auto", "token", "sequence"] = "auto",
    return_metrics: bool = False,
) -> Tensor | tuple[Tensor, PolicyLossMetrics]:
    """Clipped policy loss, with a KL term towards a reference policy.

    Per token, with ``r = exp(logprobs - old_logprobs)``, ``A`` the advantage and
    ``u = ref_logprobs - logprobs``::

        -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A) + kl_multiplier * (exp(u) - u - 1)

    ``logprobs`` (as from ``selective_log_softmax`` or
    ``chunked_linear_selective_log_softmax``; fp16, bf16 or fp32) are padded
    ``[sequences, length]`` or packed ``[tokens]`` with ``cu_seqlens``
    ``[sequences + 1]`` (int32 / int64; without it, all tokens are one sequence).
    ``mask`` (bool, like ``logprobs``) is True on the tokens that count; what the
    others hold is never used. ``old_logprobs=None`` stands for ``logprobs``
    themselves (ratio 1, with its gradient). ``advantages`` come per token or
    per sequence (``[sequences]``, padded also ``[sequences, 1]``); where packed
    tokens are as many as sequences, ``"auto"`` takes one token per sequence, and
    anything else has to say ``advantages_per``.

    ``reduction``: ``"sum"``, ``"mean"`` over the valid tokens, or
    ``"sequence_mean"``, the mean over the sequences that have valid tokens of
    the mean over each's. No valid token gives 0.

    Returns the fp32 loss, differentiable once with respect to ``logprobs``
    alone; with ``return_metrics`` also ``PolicyLossMetrics``.
    """
    _no_grad_to(old_logprobs=old_logprobs, advantages=advantages, ref_logprobs=ref_logprobs)
    loss, state = ClippedPolicyLossFunction.apply(
        logprobs, old_logprobs, advantages, ref_logprobs, mask, cu_seqlens,
        (float(clip_low), float(clip_high), float(kl_multiplier), reduction, advantages_per), torch.is_grad_enabled(),
    )
    if not return_metrics:
        return cast(Tensor, loss)
    # a copy: the state holds a value per token, which kept metrics should not
    return loss, PolicyLossMetrics(*state[:3].clone().unbind())


def preference_loss(
    logprobs: Tensor,
    ref_logprobs: Tensor | None = None,
    mask: Tensor | None = None,
    cu_seqlens: Tensor | None = None,
    beta: float = 0.1,
    loss_type: Literal["sigmoid", "hinge", "ipo"] = "sigmoid",
    label_smoothing: float = 0.0,
    margin: float = 0.0,
    length_normalized: bool = False,
    reduction: Literal["sum", "mean"] = "mean",
    return_rewards: bool = False,
) -> Tensor | tuple[Tensor, PreferenceRewards]:
    """Preference loss of paired sequences from their tokens' log-probabilities.

    The first half of the sequences are the chosen ones, the second half the
    rejected ones, in the same order. With ``s`` a sequence's sum over its valid
    tokens of ``logprobs - ref_logprobs`` (``None``: 0), divided by their number
    if ``length_normalized``, ``h = s_chosen - s_rejected`` and
    ``z = beta * h - margin``::

        sigmoid   -(1 - e) * log sigmoid(z) - e * log sigmoid(-z),  e = label_smoothing
        hinge     max(0, 1 - z)
        ipo       (h - margin - 1 / (2 * beta)) ** 2

    summed over the pairs or averaged. ``logprobs`` are padded
    ``[sequences, length]`` or packed ``[tokens]`` with ``cu_seqlens``
    ``[sequences + 1]``; ``mask`` (bool) is True on the tokens that count. A
    sequence without any has ``s = 0``.

    Returns the fp32 loss, differentiable once with respect to ``logprobs``
    alone; with ``return_rewards`` also ``PreferenceRewards``.
    """
    _no_grad_to(ref_logprobs=ref_logprobs)
    loss, state = PreferenceLossFunction.apply(
        logprobs, ref_logprobs, mask, cu_seqlens,
        (float(beta), loss_type, float(label_smoothing), float(margin), bool(length_normalized), reduction),
    )
    if not return_rewards:
        return cast(Tensor, loss)
    rewards = state[0]
    pairs = rewards.shape[0] // 2
    return loss, PreferenceRewards(rewards[:pairs], rewards[pairs:])
