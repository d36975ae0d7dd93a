"""The token losses and the gradient clipping refuse what they cannot take, before any device call."""

import math

import pytest
import torch

from greyhound_b200 import _lib
from greyhound_b200.nn.functional import clipped_policy_loss as policy
from greyhound_b200.nn.functional import preference_loss as pref
from greyhound_b200.nn.utils import clip_by_global_norm, clip_grad_norm_, global_norm

z = torch.zeros
I32 = torch.int32


@pytest.mark.parametrize(
    "args,kw,error,match",
    [
        ((z(4), z(4), z(4)), {}, ValueError, "CUDA device"),
        ((z(4), z(5), z(4)), {}, ValueError, "old_logprobs shape"),
        ((z(4), z(4), z(4)), {"ref_logprobs": z(2, 2)}, ValueError, "ref_logprobs shape"),
        ((z(4), z(4), z(4)), {"kl_multiplier": 0.1}, ValueError, "needs ref_logprobs"),
        ((z(4), z(4), z(4)), {"kl_multiplier": math.inf, "ref_logprobs": z(4)}, ValueError, "finite"),
        ((z(4), z(4), z(4)), {"clip_low": -0.1}, ValueError, "negative"),
        ((z(4), z(4), z(4)), {"clip_high": math.nan}, ValueError, "negative"),
        ((z(4), z(4), z(4)), {"reduction": "none"}, ValueError, "Unsupported reduction"),
        ((z(4), z(4), z(4)), {"advantages_per": "row"}, ValueError, "advantages_per"),
        ((z(4), z(4), z(4)), {"mask": z(4)}, TypeError, "bool mask"),
        ((z(4), z(4), z(4)), {"mask": z(3, dtype=torch.bool)}, ValueError, "mask shape"),
        ((z(2, 2), z(2, 2), z(2)), {"cu_seqlens": z(3, dtype=I32)}, ValueError, "packed"),
        ((z(4), z(4), z(4)), {"cu_seqlens": z(3)}, TypeError, "cu_seqlens"),
        ((z(4), z(4), z(4)), {"cu_seqlens": z(0, dtype=I32)}, ValueError, "cu_seqlens"),
        ((z(2, 2, 2), None, z(2)), {}, ValueError, "sequences, length"),
        ((z(4, dtype=torch.float64), None, z(4)), {}, TypeError, "logprobs dtype"),
        ((z(4, dtype=torch.int64), None, z(4)), {}, TypeError, "logprobs dtype"),
        ((z(4), z(4, requires_grad=True), z(4)), {}, ValueError, "old_logprobs.detach"),
        ((z(4), z(4), z(4, requires_grad=True)), {}, ValueError, "advantages.detach"),
        ((z(4), z(4), z(4)), {"ref_logprobs": z(4, requires_grad=True)}, ValueError, "ref_logprobs.detach"),
    ],
)
def test_policy_refusals(args, kw, error, match):
    with pytest.raises(error, match=match):
        policy(*args, **kw)


@pytest.mark.parametrize(
    "args,kw,error,match",
    [
        ((z(4, 2),), {}, ValueError, "CUDA device"),
        ((z(3, 2),), {}, ValueError, "even number"),
        ((z(4),), {}, ValueError, "need cu_seqlens"),
        ((z(4),), {"cu_seqlens": z(4, dtype=I32)}, ValueError, "even number"),
        ((z(4, 2), z(4, 3)), {}, ValueError, "ref_logprobs shape"),
        ((z(4, 2), z(4, 2, requires_grad=True)), {}, ValueError, "ref_logprobs.detach"),
        ((z(4, 2),), {"beta": 0.0}, ValueError, "beta"),
        ((z(4, 2),), {"beta": math.inf}, ValueError, "beta"),
        ((z(4, 2),), {"margin": math.nan}, ValueError, "margin"),
        ((z(4, 2),), {"loss_type": "square"}, ValueError, "loss_type"),
        ((z(4, 2),), {"label_smoothing": 1.5}, ValueError, "label_smoothing"),
        ((z(4, 2),), {"label_smoothing": 0.1, "loss_type": "ipo"}, ValueError, "label_smoothing"),
        ((z(4, 2),), {"reduction": "sequence_mean"}, ValueError, "Unsupported reduction"),
        ((z(4, 2),), {"mask": z(4, 2)}, TypeError, "bool mask"),
    ],
)
def test_preference_refusals(args, kw, error, match):
    with pytest.raises(error, match=match):
        pref(*args, **kw)


def test_clip_refusals():
    p = torch.nn.Parameter(z(3))
    p.grad = z(3)
    for f, error, match in (
        (lambda: clip_grad_norm_(p, 1.0), ValueError, "CUDA device"),
        (lambda: clip_grad_norm_([p], -1.0), ValueError, "negative"),
        (lambda: clip_grad_norm_([p], math.nan), ValueError, "negative"),
        (lambda: clip_grad_norm_([p], 1.0, norm_type=1.0), ValueError, "norm_type"),
        (lambda: global_norm([z(3)], norm_type=3.0), ValueError, "norm_type"),
        (lambda: global_norm([z(3, dtype=torch.float64)]), TypeError, "dtype"),
        (lambda: global_norm([z(3).to_sparse()]), TypeError, "layout"),
        (lambda: clip_by_global_norm([z(3)], 1.0, out=[]), ValueError, "CUDA device|outputs"),
        (lambda: clip_by_global_norm([], 1.0, out=[z(3)]), ValueError, "0 outputs"),
    ):
        with pytest.raises(error, match=match):
            f()


def test_c_entries_refuse_bad_arguments():
    import ctypes

    lib = _lib.load()
    F, B, L = _lib.GH_F32, _lib.GH_BF16, _lib.GH_I64

    def pol(dtype=F, other=F, per=0, tokens=6, cu=None, cud=0, seqs=3, low=0.2, red=1, ws=1 << 20, lp=8):
        return lib.gh_policy_loss_fwd(lp, dtype, 8, None, other, 8, per, None, tokens, cu, cud, seqs, low, 0.2, 0.0, red, 8,
                                      8, 8, 8, 8, ws, None)

    def pr(seqs=4, tokens=8, beta=0.1, kind=0, ws=1 << 20, dtype=F, other=F):
        return lib.gh_preference_loss_fwd(8, dtype, 8, other, None, tokens, None, 0, seqs, beta, 0.0, 0.0, kind, 0, 1, 8, 8, 8, 8,
                                          ws, None)

    def clip(n=(4,), dt=(F,), mx=1.0, ws=1 << 20, src=(64,), dst=(64,), norm=8):
        k = len(n)
        P = ctypes.c_void_p * k
        return lib.gh_clip_by_global_norm(P(*src), P(*dst) if dst else None, (ctypes.c_int64 * k)(*n), (ctypes.c_int * k)(*dt), k,
                                          mx, 0, norm, 8, ws, None)

    for st, error in (
        (pol(red=3), ValueError),
        (pol(low=-1.0), ValueError),
        (pol(per=5), ValueError),
        (pol(tokens=7), ValueError),
        (pol(tokens=-1), ValueError),
        (pol(seqs=0), ValueError),
        (pol(cu=8, cud=F), TypeError),
        (pol(dtype=L), TypeError),
        (pol(other=B), TypeError),
        (pol(lp=None), ValueError),
        (pol(ws=8), RuntimeError),
        (pr(seqs=3, tokens=9), ValueError),
        (pr(beta=0.0), ValueError),
        (pr(kind=7), ValueError),
        (pr(ws=8), RuntimeError),
        (pr(dtype=L), TypeError),
        (clip(mx=-1.0), ValueError),
        (clip(dt=(L,)), TypeError),
        (clip(n=(-1,)), ValueError),
        (clip(src=(None,)), ValueError),
        (clip(src=(66,), dst=(66,)), ValueError),  # not aligned to its type
        (clip(ws=8), RuntimeError),
        (clip(norm=None), ValueError),
        # outputs that overlap each other, or another input
        (clip(n=(4, 4), dt=(F, F), src=(64, 64), dst=(64, 64)), ValueError),
        (clip(n=(4, 4), dt=(F, F), src=(64, 72), dst=(64, 72)), ValueError),
        (clip(n=(4, 4), dt=(F, F), src=(64, 128), dst=(256, 72)), ValueError),
        (clip(n=(4,), dt=(F,), src=(64,), dst=(72,)), ValueError),
    ):
        with pytest.raises(error):
            _lib.check(st, "x")


def test_workspaces_are_modest():
    """Sums per warp and sequence, never per token beyond 24 bytes for 128 of them."""
    lib = _lib.load()
    assert lib.gh_policy_loss_workspace_bytes(1 << 22, 512, 2) < 1 << 20
    assert lib.gh_preference_loss_workspace_bytes(1 << 22, 512) < 1 << 20
    assert lib.gh_global_norm_workspace_bytes(10_000) < 1 << 20


@pytest.mark.parametrize("kw", [{}, {"cu_seqlens": z(3, dtype=I32)}])
def test_a_number_is_no_batch(kw):
    for f in (lambda: pref(z(()), **kw), lambda: policy(z(()), None, z(1), **kw)):
        with pytest.raises(ValueError, match="sequences, length|packed"):
            f()
