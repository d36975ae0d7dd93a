"""Gradient norm and clipping over many tensors.

``clip_grad_norm_`` has the arguments of ``torch.nn.utils.clip_grad_norm_`` and works
without a host sync, in two launches. It takes less: the 2- and the inf-norm of
dense fp16, bf16 and fp32 gradients on one CUDA device, each with memory of its own;
other norms, fp64, sparse or distributed gradients, several devices and shared
gradients are refused. ``clip_by_global_norm`` is the form for a list of tensors
that need not belong to parameters, in place or not.
"""

from __future__ import annotations

import math
from collections.abc import Iterable, Sequence

import torch
from torch import Tensor

from greyhound_b200.ops.grad_norm import clip

__all__ = ["clip_by_global_norm", "clip_grad_norm_", "global_norm"]


def _device(tensors: Sequence[Tensor]) -> torch.device:
    if tensors:
        return tensors[0].device
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def global_norm(tensors: Iterable[Tensor], norm_type: float = 2.0) -> Tensor:
    """Norm of all elements of ``tensors`` together, a 0-d fp32 tensor.

    ``norm_type`` is 2.0 or ``inf`` (the largest absolute value). Tensors are
    fp16, bf16 or fp32, on one device, mixed as they come; a tensor listed
    twice counts twice. Squares are summed in fp64.
    """
    ts = list(tensors)
    if not ts:
        return torch.zeros((), dtype=torch.float32, device=_device(ts))
    return clip(ts, None, 0.0, float(norm_type))


def clip_by_global_norm(
    tensors: Iterable[Tensor],
    max_norm: float,
    norm_type: float = 2.0,
    out: Iterable[Tensor] | None = None,
) -> tuple[list[Tensor], Tensor]:
    """``(clipped, norm)``: every tensor times ``min(1, max_norm / (norm + 1e-6))``.

    ``norm`` is ``global_norm(tensors)`` before clipping. ``out`` gives the
    tensors to write, of the same shapes and types: new ones by default, or
    ``tensors`` themselves for clipping in place, which writes nothing when the
    norm is below ``max_norm``. Outputs may not overlap themselves, each other or
    another tensor's input (``ValueError``; between views with gaps in their
    memory only the same view listed twice is noticed). A NaN norm makes every element NaN, an
    infinite one makes finite elements 0, as the formula says; an infinite
    ``max_norm`` changes nothing.
    """
    ts = list(tensors)
    if out is None:
        outs = [torch.empty_like(t, requires_grad=False) for t in ts]
    else:
        outs = list(out)
    if not ts:
        if outs:
            raise ValueError(f"expected 0 outputs, got {len(outs)}")
        return [], torch.zeros((), dtype=torch.float32, device=_device(ts))
    return outs, clip(ts, outs, float(max_norm), float(norm_type))


def clip_grad_norm_(
    parameters: Tensor | Iterable[Tensor],
    max_norm: float,
    norm_type: float = 2.0,
    error_if_nonfinite: bool = False,
    foreach: bool | None = None,
) -> Tensor:
    """Clip the gradients of ``parameters`` in place to a global norm of ``max_norm``.

    Returns the norm before clipping (0-d fp32, on the device). Parameters
    without a gradient do not count. The gradients are scaled by
    ``min(1, max_norm / (norm + 1e-6))`` computed on the device: the call does
    not synchronise, except with ``error_if_nonfinite``, which reads the norm
    and raises ``RuntimeError`` before any gradient has changed. ``foreach`` is
    accepted and makes no difference.
    Two parameters that share their gradient's memory raise ``ValueError``.
    """
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    grads = [g for p in parameters if (g := p.grad) is not None]
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=_device(grads))
    if not float(max_norm) >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if error_if_nonfinite:
        norm = clip(grads, None, 0.0, float(norm_type))
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of the gradients is {norm.item()}; they were not clipped")
    return clip(grads, grads, float(max_norm), float(norm_type))
