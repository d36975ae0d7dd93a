"""Reports of device-side problems by kernels that run at the same time on several streams."""

import pytest
import torch

from greyhound_b200 import _lib
from greyhound_b200.nn.functional import chunked_linear_selective_log_softmax, clipped_policy_loss, preference_loss
from greyhound_b200.testing import requires_gpu


@requires_gpu
@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_reports_of_two_streams_are_all_kept(monkeypatch, loss):
    """Bad offsets found by many threads, call after call, while another stream reports a bad index once."""
    monkeypatch.setattr(_lib, "raise_pending", lambda *a: None)
    S = 1 << 20
    lp = torch.zeros(S, device="cuda")
    cu = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    cu[1:] = cu[1:].view(-1, 2).flip(1).reshape(-1)  # every other one decreases
    H = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    index = torch.full((64,), 200, device="cuda")
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(one):
            torch.cuda._sleep(10_000_000)  # while the calls are queued
            for _ in range(40):
                if loss == "policy":
                    clipped_policy_loss(lp, None, lp, cu_seqlens=cu, reduction="sum", advantages_per="token")
                else:
                    preference_loss(lp, cu_seqlens=cu)
        with torch.cuda.stream(two):
            torch.cuda._sleep(10_000_000 + 120_000 * i)
            chunked_linear_selective_log_softmax(H, H, index)
        torch.cuda.synchronize()
        assert _lib.take_device_errors(0) == _lib.GH_DEV_BAD_LABEL | _lib.GH_DEV_BAD_SEQLENS, i
