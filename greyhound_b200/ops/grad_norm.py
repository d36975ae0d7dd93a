"""Global norm and clipping: custom ops, for calls that are traced.

Outside of tracing ``clip`` calls the kernels' wrapper itself (a list of
hundreds of tensors costs an op's Python layers more than the kernels take).
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from greyhound_b200 import _lib
from greyhound_b200.kernels.grad_norm import clip_tensors

__all__ = ["clip", "clip_by_global_norm_", "clip_by_global_norm_out", "global_norm"]


def _scalar(tensors: Sequence[Tensor]) -> Tensor:
    return torch.empty([], dtype=torch.float32, device=tensors[0].device)


@torch.library.custom_op("greyhound::global_norm", mutates_args=())
def global_norm(tensors: Sequence[Tensor], norm_type: float) -> Tensor:
    return clip_tensors(tensors, None, 0.0, norm_type, tensors[0].device)


@global_norm.register_fake
def _(tensors, norm_type):
    return _scalar(tensors)


@torch.library.custom_op("greyhound::clip_by_global_norm_", mutates_args=("tensors",))
def clip_by_global_norm_(tensors: Sequence[Tensor], max_norm: float, norm_type: float) -> Tensor:
    return clip_tensors(tensors, tensors, max_norm, norm_type, tensors[0].device)


@clip_by_global_norm_.register_fake
def _(tensors, max_norm, norm_type):
    return _scalar(tensors)


@torch.library.custom_op("greyhound::clip_by_global_norm_out", mutates_args=("outputs",))
def clip_by_global_norm_out(
    tensors: Sequence[Tensor], outputs: Sequence[Tensor], max_norm: float, norm_type: float
) -> Tensor:
    return clip_tensors(tensors, outputs, max_norm, norm_type, tensors[0].device)


@clip_by_global_norm_out.register_fake
def _(tensors, outputs, max_norm, norm_type):
    return _scalar(tensors)


def clip(tensors: Sequence[Tensor], outputs: Sequence[Tensor] | None, max_norm: float, norm_type: float) -> Tensor:
    """``clip_tensors`` for a list that is not empty, through a custom op where calls are recorded."""
    if _lib.untraced():
        return clip_tensors(tensors, outputs, max_norm, norm_type, tensors[0].device)
    with torch.no_grad():  # no gradient flows through a norm or a clipping
        if outputs is None:
            return global_norm(tensors, norm_type)
        if len(outputs) == len(tensors) and all(o is t for o, t in zip(outputs, tensors)):
            return clip_by_global_norm_(tensors, max_norm, norm_type)
        return clip_by_global_norm_out(tensors, outputs, max_norm, norm_type)
