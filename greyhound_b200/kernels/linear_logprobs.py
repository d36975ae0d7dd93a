"""Linear selective log-softmax on the device (sm_100a, via the C-ABI).

``logprobs = gather(log_softmax(inputs @ weight.T / temperature), index)`` and
its gradients without the ``[N, V]`` logits; the selective log-softmax of
src/greyhound/kernels/logprobs.py:131 taken from hidden states, as the chunked
linear cross-entropy takes the cross-entropy.
"""

from __future__ import annotations

import functools
import math
import os

import torch
from torch import Tensor

from greyhound_b200 import _lib
from greyhound_b200.kernels.linear_cross_entropy import chunk_size_for

__all__ = [
    "linear_logprobs",
    "linear_logprobs_backward",
    "linear_logprobs_backward_kept",
    "keeps_exponentials",
    "kept_bytes",
]

# Largest e^x buffer held from the forward to the backward. With it a step is
# three GEMMs, without it four and one chunk of logits' gradient: 8192 x 4096 x
# 128256 19.1-20.2 against 26.1 ms, with the same peak of memory (one chunk), and
# 2048 x 2048 x 100000 2.0 against 2.6 ms. 4 GiB is 16384 rows of a
# 128256-token vocabulary, twice the logits chunk of the largest heads;
# GREYHOUND_B200_LSM_KEEP_GB sets another limit.
_KEEP_BYTES = int(float(os.environ.get("GREYHOUND_B200_LSM_KEEP_GB") or 4) * (1 << 30))


def _validate(inputs: Tensor, weight: Tensor, index: Tensor, temperature: float) -> None:
    if inputs.ndim != 2 or weight.ndim != 2 or inputs.shape[1] != weight.shape[1]:
        raise ValueError(
            f"expected inputs [N, D] and weight [V, D], got {tuple(inputs.shape)} and {tuple(weight.shape)}"
        )
    if index.shape != (inputs.shape[0],):
        raise ValueError(f"expected index shape {(inputs.shape[0],)}, got {tuple(index.shape)}")
    if inputs.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"expected float16 or bfloat16 inputs, got {inputs.dtype}")
    if weight.dtype != inputs.dtype:
        raise TypeError(f"expected weight of dtype {inputs.dtype}, got {weight.dtype}")
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"expected int32 or int64 index, got {index.dtype}")
    if weight.shape[0] <= 0:
        raise ValueError("expected non-empty vocabulary dimension")
    if inputs.shape[1] <= 0 or inputs.shape[1] % 8:
        raise ValueError(f"expected a hidden size that is a positive multiple of 8, got {inputs.shape[1]}")
    if not (temperature > 0.0 and math.isfinite(temperature) and 1.0 / temperature < 1e30):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if not inputs.is_cuda or weight.device != inputs.device or index.device != inputs.device:
        raise ValueError("expected inputs, weight and index on the same CUDA device")


def _operand(t: Tensor) -> Tensor:
    """Row-major and 16-byte aligned, as the GEMM's bulk copies need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


# Sizes decide this and the workspaces' bytes; worked out once per shape (the
# backward runs on autograd's thread, where every line costs twice as much).
@functools.lru_cache(maxsize=1024)
def _chunk(N: int, D: int, V: int) -> int:
    return chunk_size_for(N, D, V, 2) if N > 0 else 1


@functools.lru_cache(maxsize=1024)
def _forward_bytes(N: int, V: int, chunk: int, keep: bool) -> int:
    return _lib.load().gh_lsm_fwd_workspace_bytes(N, V, chunk, int(keep))


@functools.lru_cache(maxsize=1024)
def _backward_bytes(N: int, D: int, V: int, chunk: int, code: int, kept: bool, fp32: bool) -> int:
    return _lib.load().gh_lsm_bwd_workspace_bytes(N, D, V, chunk, code, int(kept), int(fp32))


def kept_bytes(N: int, V: int, dtype: torch.dtype) -> int:
    """``gh_lsm_kept_bytes``, in arithmetic that symbolic sizes go through, too."""
    rows = (4 * N + 255) // 256
    beside = rows if dtype == torch.bfloat16 else (8 * N * ((V + 255) // 256) + 255) // 256 + 3 * rows
    return ((N * ((V + 7) // 8 * 8) * 2 + 255) // 256 + beside) * 256


def keeps_exponentials(inputs: Tensor, weight: Tensor) -> bool:
    """Whether the forward stores e^x for the backward: a buffer of at most 4 GiB."""
    if inputs.ndim != 2 or weight.ndim != 2:
        return False
    return inputs.shape[0] * ((weight.shape[0] + 7) // 8 * 8) * 2 <= _KEEP_BYTES


def linear_logprobs(
    inputs: Tensor,
    weight: Tensor,
    index: Tensor,
    ignore_index: int,
    temperature: float,
    want_state: bool = False,
    keep: bool = False,
) -> tuple[Tensor, Tensor | None, Tensor | None]:
    """``(logprobs [N] fp32, state [2, N] or None, kept (uint8) or None)``.

    One of the last two is what a backward needs: ``state`` (log-sum-exp in
    log2 units, log-probabilities) for ``linear_logprobs_backward``, ``kept`` for
    ``linear_logprobs_backward_kept``."""
    _validate(inputs, weight, index, temperature)
    N, D = inputs.shape
    V = weight.shape[0]
    dev = inputs.device
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "linear_selective_log_softmax")
        out = torch.empty(N, dtype=torch.float32, device=dev)
        state = torch.empty(2, N, dtype=torch.float32, device=dev) if want_state else None
        kept = torch.empty(kept_bytes(N, V, inputs.dtype), dtype=torch.uint8, device=dev) if keep else None
        if N == 0:
            return out, state, kept
        x, w, idx = _operand(inputs), _operand(weight), index.contiguous()
        chunk = _chunk(N, D, V)
        ws = _lib.workspace(_forward_bytes(N, V, chunk, keep), dev)
        st = lib.gh_lsm_fwd(
            x.data_ptr(), w.data_ptr(), idx.data_ptr(), _lib.dtype_code(idx.dtype), N, D, V,
            _lib.dtype_code(x.dtype), int(ignore_index), 1.0 / float(temperature), chunk, out.data_ptr(),
            _lib.ptr(state), _lib.ptr(kept), 0 if kept is None else kept.numel(), ws.data_ptr(), ws.numel(),
            _lib.stream_handle(dev),
        )
        _lib.check(st, "linear_selective_log_softmax")
        _lib.raise_on_status(ws, "linear_selective_log_softmax")
    return out, state, kept


def _check_grad(grad: Tensor, inputs: Tensor) -> Tensor:
    if grad.shape != (inputs.shape[0],) or grad.device != inputs.device:
        raise ValueError(
            f"expected grad shape {(inputs.shape[0],)} on {inputs.device}, got {tuple(grad.shape)} on {grad.device}"
        )
    return grad if grad.dtype is torch.float32 and grad.is_contiguous() else grad.to(torch.float32).contiguous()


def linear_logprobs_backward_kept(
    inputs: Tensor,
    weight: Tensor,
    kept: Tensor,
    grad: Tensor,
    temperature: float,
    fp32_grad_weight_accum: bool,
    want_input: bool,
    want_weight: bool,
) -> tuple[Tensor | None, Tensor | None]:
    """``(grad_input [N, D], grad_weight [V, D])`` from the stored e^x."""
    N, D = inputs.shape
    V = weight.shape[0]
    dev = inputs.device
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "linear_selective_log_softmax backward")
        x, w, g = _operand(inputs), _operand(weight), _check_grad(grad, inputs)
        gi = torch.empty_like(x) if want_input else None
        gw = torch.empty_like(w) if want_weight else None
        if N == 0:
            return gi, gw.zero_() if gw is not None else None
        chunk, code, fp32 = _chunk(N, D, V), _lib.dtype_code(x.dtype), bool(fp32_grad_weight_accum)
        ws = _lib.workspace(_backward_bytes(N, D, V, chunk, code, True, fp32), dev)
        st = lib.gh_lsm_bwd_kept(
            x.data_ptr(), w.data_ptr(), g.data_ptr(), N, D, V, code, 1.0 / float(temperature), chunk, int(fp32),
            kept.data_ptr(), kept.numel(), _lib.ptr(gi), _lib.ptr(gw), ws.data_ptr(), ws.numel(),
            _lib.stream_handle(dev),
        )
        _lib.check(st, "linear_selective_log_softmax backward")
        _lib.raise_on_status(ws, "linear_selective_log_softmax backward")
    return gi, gw


def linear_logprobs_backward(
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
) -> tuple[Tensor | None, Tensor | None]:
    """``(grad_input [N, D], grad_weight [V, D])``, the logits recomputed chunk by chunk."""
    _validate(inputs, weight, index, temperature)
    N, D = inputs.shape
    V = weight.shape[0]
    dev = inputs.device
    if state.shape != (2, N) or state.dtype != torch.float32 or state.device != dev or not state.is_contiguous():
        raise ValueError(f"expected state as a contiguous fp32 tensor of shape {(2, N)} on {dev}")
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "linear_selective_log_softmax backward")
        x, w, idx, g = _operand(inputs), _operand(weight), index.contiguous(), _check_grad(grad, inputs)
        gi = torch.empty_like(x) if want_input else None
        gw = torch.empty_like(w) if want_weight else None
        if N == 0:
            return gi, gw.zero_() if gw is not None else None
        chunk, code, fp32 = _chunk(N, D, V), _lib.dtype_code(x.dtype), bool(fp32_grad_weight_accum)
        ws = _lib.workspace(_backward_bytes(N, D, V, chunk, code, False, fp32), dev)
        st = lib.gh_lsm_bwd(
            x.data_ptr(), w.data_ptr(), idx.data_ptr(), _lib.dtype_code(idx.dtype), state.data_ptr(),
            g.data_ptr(), N, D, V, code, int(ignore_index), 1.0 / float(temperature), chunk, int(fp32),
            _lib.ptr(gi), _lib.ptr(gw), ws.data_ptr(), ws.numel(), _lib.stream_handle(dev),
        )
        _lib.check(st, "linear_selective_log_softmax backward")
        _lib.raise_on_status(ws, "linear_selective_log_softmax backward")
    return gi, gw
