"""Global norm of a list of tensors and clipping to a largest norm (sm_100a, via
the C-ABI): two launches for up to 896 tensors, whatever their sizes."""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch
from torch import Tensor

from greyhound_b200 import _lib

__all__ = ["clip_tensors", "is_dense"]


def is_dense(t: Tensor) -> bool:
    """Whether ``t`` fills its memory span without gaps or overlaps, in any order of dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _validate(tensors: Sequence[Tensor], norm_type: float) -> None:
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2.0 or inf, got {norm_type}")
    dev = tensors[0].device if tensors else None
    for i, t in enumerate(tensors):
        if t.layout != torch.strided:
            raise TypeError(f"expected dense tensors, got layout {t.layout} at {i}")
        if t.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError(f"unsupported dtype of tensor {i}: {t.dtype}")
        if not t.is_cuda or t.device != dev:
            raise ValueError(f"expected all tensors on one CUDA device, got {t.device} at {i} and {dev} before it")


def clip_tensors(
    tensors: Sequence[Tensor],
    outputs: Sequence[Tensor] | None,
    max_norm: float,
    norm_type: float,
    device: torch.device,
) -> Tensor:
    """The norm of all ``tensors`` (0-d fp32); with ``outputs``, also
    ``outputs[i] = min(1, max_norm / (norm + 1e-6)) * tensors[i]``.

    An output has its tensor's shape, type and strides; it may be the tensor."""
    _validate(tensors, norm_type)
    if outputs is not None:
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        if len(outputs) != len(tensors):
            raise ValueError(f"expected {len(tensors)} outputs, got {len(outputs)}")
        for i, (o, t) in enumerate(zip(outputs, tensors)):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device:
                raise ValueError(f"output {i} must match its tensor in shape, dtype and device")
    lib = _lib.load()
    n = len(tensors)
    with torch.cuda.device(device):
        _lib.raise_pending(device, "clip_by_global_norm")
        # a tensor with gaps, or an output laid out otherwise, goes through dense copies
        src = [t if is_dense(t) else t.contiguous() for t in tensors]
        dst = None
        if outputs is not None:
            dst = [
                o if o is t or (o.stride() == s.stride() and (s is t)) else torch.empty_like(s)
                for o, t, s in zip(outputs, tensors, src)
            ]
            dst = [s if (o is t and s is not t) else d for o, t, s, d in zip(outputs, tensors, src, dst)]
        norm = torch.empty((), dtype=torch.float32, device=device)
        ws = _lib.workspace(lib.gh_global_norm_workspace_bytes(n), device)
        pointers = ctypes.c_void_p * n
        st = lib.gh_clip_by_global_norm(
            pointers(*[t.data_ptr() for t in src]),
            None if dst is None else pointers(*[t.data_ptr() for t in dst]),
            (ctypes.c_int64 * n)(*[t.numel() for t in src]),
            (ctypes.c_int * n)(*[_lib.DTYPE_CODE[t.dtype] for t in src]),
            n, float(max_norm), int(norm_type == math.inf), norm.data_ptr(), ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream(device).cuda_stream,
        )
        _lib.check(st, "clip_by_global_norm")
        if outputs is not None and dst is not None:
            for o, d in zip(outputs, dst):
                if d is not o:
                    o.copy_(d)
    return norm
