"""What the policy and the preference loss share: the walk over sequences of tokens."""

import pytest
import torch

from greyhound_b200.nn.functional import clipped_policy_loss, preference_loss
from greyhound_b200.testing import requires_gpu


@requires_gpu
@pytest.mark.parametrize("loss", ["policy", "preference"])
@pytest.mark.parametrize("where", ["middle", "end"])
def test_a_million_empty_sequences_are_skipped(loss, where):
    """Offsets filled up to a fixed number: the same result as without them, and no warp walks them
    one by one (which took 330 ms a step)."""
    g = torch.Generator(device="cuda").manual_seed(41)
    n = torch.randint(1, 9, (4000,), device="cuda", generator=g)
    few = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), n.cumsum(0)])
    tail = 5 if where == "end" else 0  # tokens of no sequence
    T = int(few[-1]) + tail
    at = 4000 if where == "end" else 2000
    many = torch.cat([few[: at + 1], few[at].expand(1 << 20), few[at + 1 :]])
    lp = (-torch.rand(T, device="cuda", generator=g)).requires_grad_(True)

    def step(cu):
        if loss == "policy":
            y = clipped_policy_loss(lp, None, lp.detach() + 0.5, cu_seqlens=cu, reduction="sequence_mean")
        else:
            y = preference_loss(lp, cu_seqlens=cu, reduction="sum")
        return y.detach(), *torch.autograd.grad(y, lp)

    step(many)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = step(many)
    end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 50.0
    if loss == "policy":  # the pairs of the preference loss are others
        for a, b in zip(got, step(few)):
            assert torch.allclose(a, b, rtol=2.0**-21, atol=0.0)
    else:
        want_pairs = (many.numel() - 1) // 2
        d = torch.zeros(2 * want_pairs, dtype=torch.float64, device="cuda")
        seq = torch.searchsorted(many[1:], torch.arange(T - tail, device="cuda"), right=True)
        d.index_add_(0, seq, lp.detach()[: T - tail].double())
        z = 0.1 * (d[:want_pairs] - d[want_pairs:])
        want = torch.nn.functional.softplus(-z).sum()
        assert (got[0].double() - want).abs() <= 2.0**-22 * want
        slope = -0.1 * torch.sigmoid(-z)
        both = torch.cat([slope, -slope])[seq]
        assert ((got[1][: T - tail].double() - both).abs() <= 2.0**-22 * both.abs()).all()
        assert (got[1][T - tail :] == 0).all()
