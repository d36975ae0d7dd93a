"""Losses over per-token log-probabilities (sm_100a, via the C-ABI): the clipped
policy loss with a KL term, and the preference loss over pairs of sequences.

Log-probabilities are padded ``[sequences, length]`` or packed ``[tokens]`` with
offsets ``cu_seqlens``; a boolean mask may leave positions out.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch import Tensor

from greyhound_b200 import _lib

__all__ = [
    "policy_loss_forward",
    "policy_loss_backward",
    "preference_loss_forward",
    "preference_loss_backward",
    "policy_state_size",
]

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
REDUCTIONS = {"sum": 0, "mean": 1, "sequence_mean": 2}
KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}
ADVANTAGES_PER = {"token": 0, "sequence": 1, "auto": 2}


class _Layout(NamedTuple):
    tokens: int
    seqs: int
    cu: Tensor | None
    cu_code: int


def _check_like(name: str, t: Tensor, logprobs: Tensor) -> None:
    if t.shape != logprobs.shape:
        raise ValueError(f"expected {name} shape {tuple(logprobs.shape)}, got {tuple(t.shape)}")
    if t.device != logprobs.device:
        raise ValueError(f"expected {name} on {logprobs.device}, got {t.device}")


def _no_grad_to(**tensors: Tensor | None) -> None:
    for name, t in tensors.items():
        if t is not None and t.requires_grad:
            raise ValueError(f"the loss is not differentiable with respect to {name}; pass {name}.detach()")


def _layout(logprobs: Tensor, mask: Tensor | None, cu_seqlens: Tensor | None) -> _Layout:
    if logprobs.ndim not in (1, 2):
        raise ValueError(f"expected logprobs [sequences, length] or [tokens], got shape {tuple(logprobs.shape)}")
    if logprobs.dtype not in _FLOATS:
        raise TypeError(f"unsupported logprobs dtype: {logprobs.dtype}")
    if mask is not None:
        _check_like("mask", mask, logprobs)
        if mask.dtype != torch.bool:
            raise TypeError(f"expected a bool mask, got {mask.dtype}")
    if cu_seqlens is not None:
        if logprobs.ndim != 1:
            raise ValueError("cu_seqlens goes with packed logprobs [tokens]")
        if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1:
            raise ValueError(f"expected cu_seqlens [sequences + 1], got shape {tuple(cu_seqlens.shape)}")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"expected int32 or int64 cu_seqlens, got {cu_seqlens.dtype}")
        if cu_seqlens.device != logprobs.device:
            raise ValueError(f"expected cu_seqlens on {logprobs.device}, got {cu_seqlens.device}")
    if not logprobs.is_cuda:
        raise ValueError("expected logprobs on a CUDA device (greyhound_b200 has no CPU path)")
    if cu_seqlens is not None:
        return _Layout(logprobs.numel(), cu_seqlens.numel() - 1, cu_seqlens.contiguous(),
                       _lib.dtype_code(cu_seqlens.dtype))
    return _Layout(logprobs.numel(), logprobs.shape[0] if logprobs.ndim == 2 else 1, None, 0)


def _others(logprobs: Tensor, *ts: Tensor | None) -> tuple[int, list[Tensor | None]]:
    """The other log-probabilities, all in logprobs' type or all in fp32."""
    for t in ts:
        if t is not None and not t.is_floating_point():
            raise TypeError(f"unsupported log-probability dtype: {t.dtype}")
    same = all(t is None or t.dtype == logprobs.dtype for t in ts)
    dtype = logprobs.dtype if same else torch.float32
    return _lib.dtype_code(dtype), [None if t is None else t.to(dtype).contiguous() for t in ts]


def _seqs(logprobs: Tensor, cu_seqlens: Tensor | None) -> int:
    return cu_seqlens.numel() - 1 if cu_seqlens is not None else logprobs.shape[0] if logprobs.ndim == 2 else 1


@functools.lru_cache(maxsize=1024)  # sizes alone decide it
def _policy_workspace(tokens: int, seqs: int, reduction: str) -> int:
    """Floats of the policy loss's workspace, rounded to 16 bytes."""
    return (int(_lib.load().gh_policy_loss_workspace_bytes(tokens, seqs, REDUCTIONS[reduction])) + 15) // 16 * 4


@functools.lru_cache(maxsize=1024)
def _preference_workspace(tokens: int, seqs: int) -> int:
    return _lib.load().gh_preference_loss_workspace_bytes(tokens, seqs)


def policy_state_size(logprobs: Tensor, cu_seqlens: Tensor | None, reduction: str, want_grad: bool) -> int:
    tokens, seqs = int(logprobs.numel()), int(_seqs(logprobs, cu_seqlens))  # symbolic sizes become these
    return 4 + _policy_workspace(tokens, seqs, reduction) + (tokens if want_grad else 0)


def _advantages(advantages: Tensor, logprobs: Tensor, lay: _Layout, per: str) -> tuple[Tensor, int]:
    """(contiguous fp32 advantages, the C-ABI's advantages_per)."""
    if advantages.device != logprobs.device:
        raise ValueError(f"expected advantages on {logprobs.device}, got {advantages.device}")
    if not advantages.is_floating_point():
        raise TypeError(f"unsupported advantages dtype: {advantages.dtype}")
    token = advantages.shape == logprobs.shape
    if logprobs.ndim == 2:
        seq = advantages.shape in ((lay.seqs,), (lay.seqs, 1))
    else:
        seq = advantages.shape == (lay.seqs,)
    if per == "token":
        seq = False
    elif per == "sequence":
        token = False
    if not token and not seq:
        raise ValueError(
            f"expected advantages per token {tuple(logprobs.shape)} or per sequence {(lay.seqs,)}, "
            f"got {tuple(advantages.shape)}"
        )
    code = 1 if not token else 2 if seq and lay.cu is not None else 0
    return advantages.to(torch.float32).contiguous(), code


def policy_loss_forward(
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
    advantages_per: str = "auto",
    want_grad: bool = True,
) -> tuple[Tensor, Tensor]:
    """``(loss, state)``, both fp32.

    ``state`` is what ``policy_loss_backward`` needs, in one buffer: mean KL
    estimate, share of clipped tokens, valid tokens and the weight of a token
    (4), the workspace, and with ``want_grad`` the tokens' unweighted gradients.
    """
    if reduction not in REDUCTIONS:
        raise ValueError(f"Unsupported reduction: {reduction}")
    if advantages_per not in ADVANTAGES_PER:
        raise ValueError(f"advantages_per must be 'auto', 'token' or 'sequence', got {advantages_per!r}")
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError(f"clip_low and clip_high must not be negative, got {clip_low} and {clip_high}")
    if not math.isfinite(kl_multiplier):
        raise ValueError(f"kl_multiplier must be finite, got {kl_multiplier}")
    if kl_multiplier != 0.0 and ref_logprobs is None:
        raise ValueError("kl_multiplier needs ref_logprobs")
    for name, t in (("old_logprobs", old_logprobs), ("ref_logprobs", ref_logprobs)):
        if t is not None:
            _check_like(name, t, logprobs)
    lay = _layout(logprobs, mask, cu_seqlens)
    adv, per = _advantages(advantages, logprobs, lay, advantages_per)
    other, (old, ref) = _others(logprobs, old_logprobs, ref_logprobs)
    dev = logprobs.device
    red = REDUCTIONS[reduction]
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "clipped_policy_loss")
        lp = logprobs.contiguous()
        m = None if mask is None else mask.contiguous()
        loss = torch.empty((), dtype=torch.float32, device=dev)
        ws = _policy_workspace(lay.tokens, lay.seqs, reduction)
        state = torch.empty(4 + ws + (lay.tokens if want_grad else 0), dtype=torch.float32, device=dev)
        at = state.data_ptr()
        st = lib.gh_policy_loss_fwd(
            lp.data_ptr(), _lib.dtype_code(lp.dtype), _lib.ptr(old), _lib.ptr(ref), other, adv.data_ptr(), per,
            _lib.ptr(m), lay.tokens, _lib.ptr(lay.cu), lay.cu_code, lay.seqs, float(clip_low), float(clip_high),
            float(kl_multiplier), red, loss.data_ptr(), at, at + 16 + 4 * ws if want_grad else None, at + 12,
            at + 16, 4 * ws, _lib.stream_handle(dev),
        )
        _lib.check(st, "clipped_policy_loss")
        _lib.raise_on_report(dev, "clipped_policy_loss")
    return loss, state


def policy_loss_backward(
    state: Tensor,
    cu_seqlens: Tensor | None,
    grad_output: Tensor,
    shape: list[int] | torch.Size,
    dtype: torch.dtype,
    reduction: str,
) -> Tensor:
    """``grad_output * dloss/dlogprobs`` in ``shape`` and ``dtype``."""
    # runs on autograd's thread, where every line costs more than in the forward
    dev = state.device
    tokens = math.prod(shape)
    seqs = cu_seqlens.numel() - 1 if cu_seqlens is not None else shape[0] if len(shape) == 2 else 1
    ws = state.numel() - 4 - tokens
    if ws < 0:
        raise ValueError("the state does not belong to a forward of this shape with gradients")
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "clipped_policy_loss backward")
        grad = torch.empty(shape, dtype=dtype, device=dev)
        g = grad_output if grad_output.dtype == torch.float32 else grad_output.to(torch.float32)
        at = state.data_ptr()
        st = _lib.load().gh_policy_loss_bwd(
            at + 16 + 4 * ws, at + 12, at + 16, 4 * ws, g.data_ptr(), tokens, _lib.ptr(cu_seqlens),
            0 if cu_seqlens is None else _lib.DTYPE_CODE[cu_seqlens.dtype], seqs, REDUCTIONS[reduction],
            grad.data_ptr(), _lib.DTYPE_CODE[dtype], _lib.stream_handle(dev),
        )
        _lib.check(st, "clipped_policy_loss backward")
    return grad


def preference_loss_forward(
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
    """``(loss, state [2, sequences])``, fp32: rewards, and the gradient of a valid token of each sequence."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"Unsupported reduction: {reduction}")
    if loss_type not in KINDS:
        raise ValueError(f"loss_type must be 'sigmoid', 'hinge' or 'ipo', got {loss_type!r}")
    if not (beta > 0.0 and math.isfinite(beta)):
        raise ValueError(f"beta must be positive and finite, got {beta}")
    if not math.isfinite(margin):
        raise ValueError(f"margin must be finite, got {margin}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must lie in [0, 1], got {label_smoothing}")
    if label_smoothing != 0.0 and loss_type != "sigmoid":
        raise ValueError("label_smoothing goes with loss_type='sigmoid'")
    if ref_logprobs is not None:
        _check_like("ref_logprobs", ref_logprobs, logprobs)
    if logprobs.ndim == 0:
        raise ValueError("expected logprobs [sequences, length] or [tokens], got shape ()")
    if logprobs.ndim == 1 and cu_seqlens is None:
        raise ValueError("packed logprobs need cu_seqlens")
    seqs = cu_seqlens.numel() - 1 if cu_seqlens is not None and cu_seqlens.ndim == 1 else logprobs.shape[0]
    if seqs % 2:
        raise ValueError(f"expected an even number of sequences (the chosen, then the rejected ones), got {seqs}")
    lay = _layout(logprobs, mask, cu_seqlens)
    other, (ref,) = _others(logprobs, ref_logprobs)
    dev = logprobs.device
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "preference_loss")
        lp = logprobs.contiguous()
        m = None if mask is None else mask.contiguous()
        loss = torch.empty((), dtype=torch.float32, device=dev)
        state = torch.empty(2, lay.seqs, dtype=torch.float32, device=dev)
        at = state.data_ptr()
        ws = _lib.workspace(_preference_workspace(lay.tokens, lay.seqs), dev)
        st = lib.gh_preference_loss_fwd(
            lp.data_ptr(), _lib.dtype_code(lp.dtype), _lib.ptr(ref), other, _lib.ptr(m), lay.tokens,
            _lib.ptr(lay.cu), lay.cu_code, lay.seqs, float(beta), float(margin), float(label_smoothing),
            KINDS[loss_type], int(length_normalized), int(reduction == "mean"), loss.data_ptr(), at,
            at + 4 * lay.seqs, ws.data_ptr(), ws.numel(), _lib.stream_handle(dev),
        )
        _lib.check(st, "preference_loss")
        _lib.raise_on_report(dev, "preference_loss")
    return loss, state


def preference_loss_backward(
    state: Tensor,
    grad_output: Tensor,
    mask: Tensor | None,
    cu_seqlens: Tensor | None,
    shape: list[int] | torch.Size,
    dtype: torch.dtype,
) -> Tensor:
    """``grad_output * dloss/dlogprobs`` in ``shape`` and ``dtype``."""
    dev = state.device
    seqs = state.shape[1]
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.raise_pending(dev, "preference_loss backward")
        grad = torch.empty(shape, dtype=dtype, device=dev)
        g = grad_output.to(torch.float32)
        m = None if mask is None else mask.contiguous()
        cu = None if cu_seqlens is None else cu_seqlens.contiguous()
        st = lib.gh_preference_loss_bwd(
            state.data_ptr() + 4 * seqs, g.data_ptr(), _lib.ptr(m), grad.numel(), _lib.ptr(cu),
            0 if cu is None else _lib.dtype_code(cu.dtype), seqs, grad.data_ptr(), _lib.dtype_code(dtype),
            _lib.stream_handle(dev),
        )
        _lib.check(st, "preference_loss backward")
    return grad
