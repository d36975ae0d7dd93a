"""chunked_linear_selective_log_softmax refuses what it cannot take, before any
device call; the buffer sizes of its passes."""

import pytest
import torch

from greyhound_b200 import _lib
from greyhound_b200.kernels.linear_logprobs import kept_bytes
from greyhound_b200.nn.functional import chunked_linear_selective_log_softmax as f

BF = torch.bfloat16


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize(
    "args,kw,error,match",
    [
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int64)), {}, ValueError, "same CUDA device"),
        ((z(4, 16), z(9, 24), z(4, dtype=torch.int64)), {}, ValueError, "expected inputs"),
        ((z(4, 16), z(16), z(4, dtype=torch.int64)), {}, ValueError, "expected inputs"),
        ((z(4, 16), z(9, 16), z(5, dtype=torch.int64)), {}, ValueError, "index shape"),
        ((z(4, 16), z(9, 16), z(4, 1, dtype=torch.int64)), {}, ValueError, "index shape"),
        ((z(4, 16, dtype=torch.float32), z(9, 16, dtype=torch.float32), z(4, dtype=torch.int64)), {}, TypeError, "float16 or bfloat16"),
        ((z(4, 16), z(9, 16, dtype=torch.float16), z(4, dtype=torch.int64)), {}, TypeError, "weight of dtype"),
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int16)), {}, TypeError, "int32 or int64"),
        ((z(4, 12), z(9, 12), z(4, dtype=torch.int64)), {}, ValueError, "multiple of 8"),
        ((z(4, 0), z(9, 0), z(4, dtype=torch.int64)), {}, ValueError, "multiple of 8"),
        ((z(4, 16), z(0, 16), z(4, dtype=torch.int64)), {}, ValueError, "non-empty vocabulary"),
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int64)), {"temperature": 0.0}, ValueError, "temperature"),
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int64)), {"temperature": float("nan")}, ValueError, "temperature"),
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int64)), {"temperature": float("inf")}, ValueError, "temperature"),
        ((z(4, 16), z(9, 16), z(4, dtype=torch.int64)), {"grad_weight_accum_dtype": "bf16"}, ValueError, "grad_weight_accum"),
    ],
)
def test_refusals(args, kw, error, match):
    with pytest.raises(error, match=match):
        f(*args, **kw)


def test_c_entries_refuse_bad_arguments():
    lib = _lib.load()
    BFC, F16, I64 = _lib.GH_BF16, _lib.GH_F16, _lib.GH_I64

    def fwd(dtype=BFC, D=16, kept=None, kb=0, wb=1 << 30, inv_t=1.0, idt=I64, H=16, W=16, ws=16):
        return lib.gh_lsm_fwd(H, W, 8, idt, 4, D, 9, dtype, -100, inv_t, 4, 8, None, kept, kb, ws, wb, None)

    def kept_bwd(dtype=BFC, wb=1 << 30, H=16, gi=16, gw=16, kept=16, kb=1 << 20):
        return lib.gh_lsm_bwd_kept(H, 16, 8, 4, 16, 9, dtype, 1.0, 4, 1, kept, kb, gi, gw, 16, wb, None)

    def bwd(index=8, wb=1 << 30, W=16, gi=16):
        return lib.gh_lsm_bwd(16, W, index, I64, 8, 8, 4, 16, 9, BFC, -100, 1.0, 4, 1, gi, 16, 16, wb, None)

    for st, error in (
        (fwd(dtype=_lib.GH_F32), TypeError),
        (fwd(idt=_lib.GH_F32), TypeError),
        (fwd(D=12), ValueError),
        (fwd(inv_t=0.0), ValueError),
        (fwd(wb=16), RuntimeError),
        (fwd(kept=16, kb=16), RuntimeError),
        (fwd(dtype=F16, kept=16, kb=64), RuntimeError),
        (fwd(H=8), ValueError),
        (fwd(W=2), ValueError),
        (fwd(ws=8), ValueError),
        (fwd(H=None), ValueError),
        (kept_bwd(dtype=F16, kb=64), RuntimeError),
        (kept_bwd(dtype=F16, wb=64), RuntimeError),
        (kept_bwd(wb=16), RuntimeError),
        (kept_bwd(kb=16), RuntimeError),
        (kept_bwd(H=8), ValueError),
        (kept_bwd(gi=8), ValueError),
        (kept_bwd(gw=2), ValueError),
        (bwd(index=None), ValueError),
        (bwd(wb=16), RuntimeError),
        (bwd(W=4), ValueError),
        (bwd(gi=4), ValueError),
    ):
        with pytest.raises(error):
            _lib.check(st, "x")


def test_buffer_sizes():
    """Stored e^x is 2 bytes a logit; the forward without it, and the
    recomputed backward, do not grow with N * V."""
    lib = _lib.load()
    for n, v in ((1, 1), (7, 9), (64, 100), (65, 128256), (16384, 131072)):
        assert kept_bytes(n, v, torch.bfloat16) == lib.gh_lsm_kept_bytes(n, v, _lib.GH_BF16)
        assert kept_bytes(n, v, torch.float16) == lib.gh_lsm_kept_bytes(n, v, _lib.GH_F16)
    assert lib.gh_lsm_kept_bytes(8192, 128256, _lib.GH_F16) < 8192 * 128256 * 2 + (64 << 20)
    assert lib.gh_lsm_kept_bytes(8192, 128256, _lib.GH_BF16) < 8192 * 128256 * 2 + (1 << 20)
    assert lib.gh_lsm_fwd_workspace_bytes(65536, 128256, 8192, 0) < 64 << 20
    assert lib.gh_lsm_bwd_workspace_bytes(65536, 4096, 128256, 8192, _lib.GH_BF16, 0, 1) < (2 << 30) + 4 * 4096 * 128256 + (256 << 20)
