"""Linear selective log-softmax custom ops + autograd Function.

The forward is one of two ops: ``greyhound::linear_selective_log_softmax_kept``
stores e^x in 16 bits for a backward of two GEMMs;
``greyhound::linear_selective_log_softmax`` returns the per-row log-sum-exp,
from which the backward recomputes the logits chunk by chunk. Without a
gradient to come, the second runs and stores nothing per vocabulary entry.
"""

from __future__ import annotations

from typing import Any

import torch
from torch import Tensor

from greyhound_b200 import _lib
from greyhound_b200.kernels.linear_logprobs import (
    keeps_exponentials,
    kept_bytes,
    linear_logprobs,
    linear_logprobs_backward,
    linear_logprobs_backward_kept,
)

__all__ = [
    "ChunkedLinearSelectiveLogSoftmaxFunction",
    "linear_selective_log_softmax",
    "linear_selective_log_softmax_bwd",
    "linear_selective_log_softmax_kept",
    "linear_selective_log_softmax_kept_bwd",
]


def _rows(inputs: Tensor) -> Tensor:
    return torch.empty([inputs.shape[0]], dtype=torch.float32, device=inputs.device)


def _grads(inputs: Tensor, weight: Tensor, want_input: bool, want_weight: bool) -> tuple[Tensor, Tensor]:
    return (
        inputs.new_empty(inputs.shape if want_input else (0,)),
        weight.new_empty(weight.shape if want_weight else (0,)),
    )


def _present(gi: Tensor | None, gw: Tensor | None, inputs: Tensor, weight: Tensor) -> tuple[Tensor, Tensor]:
    # ops return tensors; an unwanted gradient is an empty one
    return (inputs.new_empty(0) if gi is None else gi, weight.new_empty(0) if gw is None else gw)


@torch.library.custom_op("greyhound::linear_selective_log_softmax", mutates_args=())
def linear_selective_log_softmax(
    inputs: Tensor,  # [N, D]
    weight: Tensor,  # [V, D]
    index: Tensor,  # [N]
    ignore_index: int,
    temperature: float,
) -> tuple[Tensor, Tensor]:
    """(logprobs [N], state [2, N]: log-sum-exp in log2 units, log-probabilities)."""
    out, state, _ = linear_logprobs(inputs, weight, index, ignore_index, temperature, want_state=True)
    assert state is not None
    return out, state


@linear_selective_log_softmax.register_fake
def _(inputs, weight, index, ignore_index, temperature):
    return _rows(inputs), torch.empty([2, inputs.shape[0]], dtype=torch.float32, device=inputs.device)


@torch.library.custom_op("greyhound::linear_selective_log_softmax_kept", mutates_args=())
def linear_selective_log_softmax_kept(
    inputs: Tensor,
    weight: Tensor,
    index: Tensor,
    ignore_index: int,
    temperature: float,
) -> tuple[Tensor, Tensor]:
    """(logprobs [N], stored e^x and row factors (uint8))."""
    out, _, kept = linear_logprobs(inputs, weight, index, ignore_index, temperature, keep=True)
    assert kept is not None
    return out, kept


@linear_selective_log_softmax_kept.register_fake
def _(inputs, weight, index, ignore_index, temperature):
    kept = torch.empty(kept_bytes(inputs.shape[0], weight.shape[0], inputs.dtype), dtype=torch.uint8, device=inputs.device)
    return _rows(inputs), kept


@torch.library.custom_op("greyhound::linear_selective_log_softmax_bwd", mutates_args=())
def linear_selective_log_softmax_bwd(
    inputs: Tensor,
    weight: Tensor,
    index: Tensor,
    state: Tensor,
    grad: Tensor,
    ignore_index: int,
    temperature: float,
    fp32_grad_weight_accum: bool,
    want_input: bool,
    want_weight: bool,
) -> tuple[Tensor, Tensor]:
    """(grad_input [N, D], grad_weight [V, D]); an unwanted one is empty."""
    gi, gw = linear_logprobs_backward(
        inputs, weight, index, state, grad, ignore_index, temperature, fp32_grad_weight_accum, want_input,
        want_weight,
    )
    return _present(gi, gw, inputs, weight)


@linear_selective_log_softmax_bwd.register_fake
def _(inputs, weight, index, state, grad, ignore_index, temperature, fp32_grad_weight_accum, want_input, want_weight):
    return _grads(inputs, weight, want_input, want_weight)


@torch.library.custom_op("greyhound::linear_selective_log_softmax_kept_bwd", mutates_args=())
def linear_selective_log_softmax_kept_bwd(
    inputs: Tensor,
    weight: Tensor,
    kept: Tensor,
    grad: Tensor,
    temperature: float,
    fp32_grad_weight_accum: bool,
    want_input: bool,
    want_weight: bool,
) -> tuple[Tensor, Tensor]:
    """(grad_input [N, D], grad_weight [V, D]); an unwanted one is empty."""
    gi, gw = linear_logprobs_backward_kept(
        inputs, weight, kept, grad, temperature, fp32_grad_weight_accum, want_input, want_weight
    )
    return _present(gi, gw, inputs, weight)


@linear_selective_log_softmax_kept_bwd.register_fake
def _(inputs, weight, kept, grad, temperature, fp32_grad_weight_accum, want_input, want_weight):
    return _grads(inputs, weight, want_input, want_weight)


class ChunkedLinearSelectiveLogSoftmaxFunction(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any,
        inputs: Tensor,  # [N, D]
        weight: Tensor,  # [V, D]
        index: Tensor,  # [N]
        ignore_index: int = -100,
        temperature: float = 1.0,
        fp32_grad_weight_accum: bool = True,
        grad_enabled: bool = True,  # the caller's mode: in here gradients are always off
    ) -> Tensor:
        plain = _lib.eager(inputs) and _lib.eager(weight)
        if not grad_enabled or not (ctx.needs_input_grad[0] or ctx.needs_input_grad[1]):
            if plain:
                return linear_logprobs(inputs, weight, index, ignore_index, temperature)[0]
            return linear_selective_log_softmax(inputs, weight, index, ignore_index, temperature)[0]
        ctx.temperature, ctx.fp32_accum = temperature, fp32_grad_weight_accum
        ctx.kept = keeps_exponentials(inputs, weight)
        if ctx.kept:
            if plain:
                out, _, kept = linear_logprobs(inputs, weight, index, ignore_index, temperature, keep=True)
            else:
                out, kept = linear_selective_log_softmax_kept(inputs, weight, index, ignore_index, temperature)
            ctx.save_for_backward(inputs, weight, kept)
            return out
        if plain:
            out, state, _ = linear_logprobs(inputs, weight, index, ignore_index, temperature, want_state=True)
        else:
            out, state = linear_selective_log_softmax(inputs, weight, index, ignore_index, temperature)
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(inputs, weight, index, state)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad: Tensor):  # type: ignore[override]
        want = ctx.needs_input_grad
        if ctx.kept:
            inputs, weight, kept = ctx.saved_tensors
            bwd = linear_logprobs_backward_kept if _lib.eager(grad) else linear_selective_log_softmax_kept_bwd
            gi, gw = bwd(
                inputs, weight, kept, grad, ctx.temperature, ctx.fp32_accum, want[0], want[1]
            )
        else:
            inputs, weight, index, state = ctx.saved_tensors
            bwd = linear_logprobs_backward if _lib.eager(grad) else linear_selective_log_softmax_bwd
            gi, gw = bwd(
                inputs, weight, index, state, grad, ctx.ignore_index, ctx.temperature, ctx.fp32_accum, want[0], want[1]
            )
        return gi if want[0] else None, gw if want[1] else None, None, None, None, None, None
