"""Global norm of a list of tensors and clipping to a largest norm (sm_100a, via
the C-ABI): two launches for up to 896 tensors, whatever their sizes."""

from __future__ import annotations

import math
import operator
from array import array
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


def _apart(t: Tensor) -> bool:
    """Whether each of ``t``'s elements has memory of its own (seen from the strides, in any order)."""
    end = 0
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride <= end:
            return False
        end += stride * (size - 1)
    return True


_CODES = {torch.float16: _lib.GH_F16, torch.bfloat16: _lib.GH_BF16, torch.float32: _lib.GH_F32}


_dtype, _layout, _shape = (operator.attrgetter(name) for name in ("dtype", "layout", "shape"))


def _on(tensors: Sequence[Tensor], index: int | None) -> bool:
    """Whether all are dense tensors on CUDA device ``index``."""
    return set(map(_layout, tensors)) <= {torch.strided} and set(map(Tensor.get_device, tensors)) <= {index}


def _dense(t: Tensor) -> Tensor:
    return t if is_dense(t) else t.detach().contiguous()


def _refuse(i: int, t: Tensor, dev: torch.device) -> None:
    if t.layout != torch.strided:
        raise TypeError(f"expected dense tensors, got layout {t.layout} at {i}")
    if t.dtype not in _CODES:
        raise TypeError(f"unsupported dtype of tensor {i}: {t.dtype}")
    raise ValueError(f"expected all tensors on one CUDA device, got {t.device} at {i} and {dev} before it")


def _operands(
    tensors: Sequence[Tensor], outputs: Sequence[Tensor] | None, device: torch.device
) -> tuple[array, Sequence[Tensor], Sequence[Tensor] | None, list[tuple[Tensor, Tensor]]]:
    """(dtype codes, dense inputs, dense outputs, copies to make afterwards)."""
    # Contiguous tensors on one device, the common list of hundreds: walked by
    # map over the tensors' methods, which costs less than half of a loop
    # (144 tensors and outputs: 100 us of host time).
    index = device.index if device.type == "cuda" else None
    dtypes = list(map(_dtype, tensors))
    found = list(map(_CODES.get, dtypes))
    if index is None or None in found or not _on(tensors, index):
        for i, t in enumerate(tensors):
            if t.dtype not in _CODES or t.device != device or t.layout != torch.strided or not t.is_cuda:
                _refuse(i, t, device)
    codes = array("i", found)
    whole = all(map(Tensor.is_contiguous, tensors))
    if outputs is None:
        return codes, tensors if whole else [_dense(t) for t in tensors], None, []
    if all(map(operator.is_, tensors, outputs)):
        outputs = tensors
    elif (
        list(map(_dtype, outputs)) != dtypes
        or list(map(_shape, outputs)) != list(map(_shape, tensors))
        or not _on(outputs, index)
    ):
        for i, (o, t) in enumerate(zip(outputs, tensors)):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device or o.layout != torch.strided:
                raise ValueError(f"output {i} must match its tensor in shape, dtype and device")
    if whole and (outputs is tensors or all(map(Tensor.is_contiguous, outputs))):
        return codes, tensors, outputs, []
    src, dst = [], []
    back: list[tuple[Tensor, Tensor]] = []
    seen: dict[tuple, int] = {}  # views with gaps: the C entry compares those without
    for i, (o, t) in enumerate(zip(outputs, tensors)):
        if o.numel() > 0 and not is_dense(o):
            if not _apart(o):
                raise ValueError(f"output {i} has elements that share memory")
            j = seen.setdefault((o.data_ptr(), o.dtype, o.shape, o.stride()), i)
            if j != i:
                raise ValueError(f"tensors {j} and {i} share memory that would be scaled twice")
        s = _dense(t)
        # written in place of the input's dense copy, or where input and output are laid out alike
        d = s if o is t else o if s is t and o.stride() == t.stride() else torch.empty_like(s)
        src.append(s)
        dst.append(d)
        if d is not o:
            back.append((o, d))
    return codes, src, dst, back


def clip_tensors(
    tensors: Sequence[Tensor],
    outputs: Sequence[Tensor] | None,
    max_norm: float,
    norm_type: float,
    device: torch.device,
) -> Tensor:
    """The norm of all ``tensors`` (0-d fp32); with ``outputs``, also
    ``outputs[i] = min(1, max_norm / (norm + 1e-6)) * tensors[i]``.

    An output has its tensor's shape and type; it may be the tensor itself."""
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type must be 2.0 or inf, got {norm_type}")
    if outputs is not None:
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        if len(outputs) != len(tensors):
            raise ValueError(f"expected {len(tensors)} outputs, got {len(outputs)}")
    codes, src, dst, back = _operands(tensors, outputs, device)
    lib = _lib.load()
    n = len(src)
    with _lib.on_device(device):
        _lib.raise_pending(device, "clip_by_global_norm")
        norm = torch.empty((), dtype=torch.float32, device=device)
        ws = _lib.workspace(lib.gh_global_norm_workspace_bytes(n), device)
        ins = array("Q", map(Tensor.data_ptr, src))
        if 0 in ins:  # empty ones, or wrappers around other tensors
            for i, t in enumerate(src):
                if ins[i] == 0 and t.numel() > 0:
                    raise TypeError(f"tensor {i} ({type(t).__name__}) has no memory of its own; pass its local tensor")
        outs = None if dst is None else ins if dst is src else array("Q", map(Tensor.data_ptr, dst))
        sizes = array("q", map(Tensor.numel, src))
        st = lib.gh_clip_by_global_norm(
            ins.buffer_info()[0], None if outs is None else outs.buffer_info()[0], sizes.buffer_info()[0],
            codes.buffer_info()[0], n, float(max_norm), int(norm_type == math.inf), norm.data_ptr(), ws.data_ptr(),
            ws.numel(), _lib.stream_handle(device),
        )
        _lib.check(st, "clip_by_global_norm")
        if outputs is not None:
            try:  # what autograd saved of them is no longer what it was
                torch.autograd.graph.increment_version(outputs)
            except RuntimeError:  # inference tensors keep no count
                pass
        for o, d in back:
            o.detach().copy_(d)
    return norm
