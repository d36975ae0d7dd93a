"""preference_loss against its formula in 64 bits.

Tolerances: differences, sums and the pairs' terms are fp64 from exact fp32 or
16-bit inputs; each result is rounded to fp32 once, a gradient a second time
(times grad_output) and to the log-probabilities' type. 2^-23 of a result, and half
a step of the gradient's type, hold that; sums of n terms in fp64 add
n 2^-53 of their absolute sum.
"""

import math

import pytest
import torch
from _token_batches import HALF, batch
from torch.library import opcheck

from greyhound_b200 import _lib
from greyhound_b200.nn.functional import preference_loss
from greyhound_b200.ops.token_losses import preference_loss_bwd, preference_loss_fwd
from greyhound_b200.testing import requires_gpu

R = 2.0**-23


def reference(lp, ref, valid, seq, S, beta, kind, smooth, margin, normalized, mean):
    """(loss, per-sequence rewards, gradient) over flat tokens, by autograd in 64 bits."""
    lp = torch.where(valid, lp.double(), 0.0).requires_grad_(True)
    diff = lp if ref is None else lp - torch.where(valid, ref.double(), 0.0)
    n = torch.zeros(S, dtype=torch.float64, device=lp.device).index_add(0, seq[valid], torch.ones_like(diff)[valid])
    s = torch.zeros(S, dtype=torch.float64, device=lp.device).index_add(0, seq[valid], diff[valid])
    if normalized:
        s = s / n.clamp(min=1)
    h = s[: S // 2] - s[S // 2 :]
    z = beta * h - margin
    if kind == "sigmoid":
        l = -(1 - smooth) * torch.nn.functional.logsigmoid(z) - smooth * torch.nn.functional.logsigmoid(-z)
    elif kind == "hinge":
        l = (1 - z).clamp(min=0)
    else:
        l = (h - margin - 1 / (2 * beta)) ** 2
    loss = l.sum() / (max(S // 2, 1) if mean else 1)
    (grad,) = torch.autograd.grad(loss, lp) if S else (torch.zeros_like(lp),)
    return loss.detach(), (beta * s).detach(), grad


def check(b, beta=0.1, kind="sigmoid", smooth=0.0, margin=0.0, normalized=False, reduction="mean", ref=True, grad_output=1.0):
    lp = b["lp"].clone().requires_grad_(True)
    loss, rewards = preference_loss(lp, b["ref"] if ref else None, b["mask"], b["cu"], beta, kind, smooth, margin,
                                    normalized, reduction, return_rewards=True)
    (grad,) = torch.autograd.grad(loss, lp, torch.tensor(grad_output, device="cuda"))
    flat = lambda t: t.reshape(-1)  # noqa: E731
    valid = flat(b["mask"])
    rl, rr, rg = reference(flat(b["lp"]), flat(b["ref"]) if ref else None, valid, flat(b["seq"]), b["S"], beta, kind, smooth,
                           margin, normalized, reduction == "mean")
    assert grad.shape == b["lp"].shape and grad.dtype == b["lp"].dtype and loss.dtype == torch.float32
    slack = 2.0**-40  # fp64 sums of up to 2^13 terms' worth of cancellation
    assert (loss.double() - rl).abs() <= R * rl.abs() + slack * (1 + rl.abs())
    got = torch.cat([rewards.chosen, rewards.rejected]).double()
    assert ((got - rr).abs() <= R * rr.abs() + slack).all()
    rg = rg * grad_output
    tiny = torch.finfo(grad.dtype).smallest_normal * HALF[grad.dtype] * 2
    err = (flat(grad).double() - rg).abs()
    assert (err <= (R + HALF[grad.dtype]) * rg.abs() + tiny + slack * rg.abs().amax().clamp(max=1)).all(), err.max()
    assert (flat(grad)[~valid] == 0).all()
    return loss.detach(), grad


KINDS = [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)]


@requires_gpu
@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("kind,smooth", KINDS)
@pytest.mark.parametrize("lengths", [[1, 1], [0, 5], [33, 0, 0, 64, 31, 1], [300, 5, 129, 1000], [1] * 40], ids=lambda x: f"{len(x)}x{max(x)}")
def test_against_formula(lengths, kind, smooth, padded):
    b = batch(lengths, torch.float32, len(lengths) * 17 + max(lengths), padded, pad=3, front=2, back=5)
    for normalized in (False, True):
        for reduction in ("mean", "sum"):
            check(b, 0.1, kind, smooth, 0.0, normalized, reduction)
    check(b, 0.7, kind, smooth, 0.3, ref=False, grad_output=-3.0)


@requires_gpu
@pytest.mark.parametrize("lengths", [[9000, 1, 0, 3333], [40] * 700, [100_000, 3], [5, 120_000, 70_001, 0]])
@pytest.mark.parametrize("padded", [True, False])
def test_many_blocks(lengths, padded):
    if padded and len(lengths) * max(lengths) > 400_000:
        lengths = lengths[:2]
    b = batch(lengths, torch.float32, 3, padded, front=9, back=700)
    check(b)
    check(b, normalized=True, kind="ipo")


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("other", [None, torch.float32])
def test_types(dtype, other):
    check(batch([300, 5, 129, 1000], dtype, 4, False, other=other), normalized=True)


@requires_gpu
@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("n", [100, 20_000])
def test_nothing_valid(padded, n):
    """Pairs whose sequences are all left out stand at z = -margin."""
    b = batch([n, 0, 3, 4], torch.float32, 6, padded, left_out=1.1)
    for normalized in (False, True):
        _, grad = check(b, normalized=normalized)
        assert (grad == 0).all()


@requires_gpu
@pytest.mark.parametrize("shape,cu", [((0,), [0]), ((5,), [3]), ((0,), [0, 0, 0]), ((0, 5), None), ((4, 0), None)])
def test_no_tokens(shape, cu):
    lp = torch.zeros(shape, device="cuda", requires_grad=True)
    c = None if cu is None else torch.tensor(cu, device="cuda", dtype=torch.int32)
    pairs = (len(cu) - 1 if cu else shape[0]) // 2
    loss, rewards = preference_loss(lp, None, cu_seqlens=c, return_rewards=True)
    (g,) = torch.autograd.grad(loss, lp)
    assert abs(loss.item() - (0.6931471805599453 if pairs else 0.0)) <= R
    assert rewards.chosen.shape == (pairs,) and (g == 0).all()


@requires_gpu
def test_far_margins():
    """z of about +-1000: softplus and sigmoid without overflow, and the gradient's limits."""
    b = batch([50, 50], torch.float32, 8, True, left_out=0.0)
    for sign in (1.0, -1.0):
        b["lp"] = torch.tensor([[20.0 * sign], [0.0]], device="cuda").expand(2, 50).contiguous()
        b["ref"] = torch.zeros_like(b["lp"])
        check(b, beta=1.0)
        check(b, beta=1.0, smooth=0.1)


@requires_gpu
def test_nan_stays_in_its_pair():
    b = batch([20, 30, 20, 30], torch.float32, 9, True, left_out=0.0)
    b["mask"] = torch.arange(30, device="cuda") < torch.tensor([20, 30, 20, 30], device="cuda")[:, None]
    b["lp"][1, 3] = float("nan")
    for kind, _ in KINDS:
        lp = b["lp"].clone().requires_grad_(True)
        loss = preference_loss(lp, b["ref"], b["mask"], loss_type=kind)
        (g,) = torch.autograd.grad(loss, lp)
        assert loss.isnan() and g[1].isnan().all() and g[3].isnan().all()
        assert torch.isfinite(g[0]).all() and torch.isfinite(g[2]).all()


@requires_gpu
@pytest.mark.parametrize("T", [60, 30_000])
@pytest.mark.parametrize("cu", [[0, 20, 10], [-5, 20, 40], [0, 20, 1 << 40], [50, 30, 0]])
def test_bad_offsets_are_reported(T, cu):
    lp = torch.randn(T, device="cuda", requires_grad=True)
    loss = preference_loss(lp, None, cu_seqlens=torch.tensor(cu, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="offsets"):
        loss.backward()
    loss.backward()
    torch.cuda.synchronize()
    assert _lib.take_device_errors(0) == 0


@requires_gpu
def test_against_differences():
    b = batch([30, 12, 25, 14], torch.float32, 10, True)
    _, grad = check(b, 0.3, "sigmoid", 0.1, 0.2)
    flat = lambda t: t.reshape(-1)  # noqa: E731
    f = lambda x: reference(flat(x), flat(b["ref"]), flat(b["mask"]), flat(b["seq"]), 4, 0.3, "sigmoid", 0.1, 0.2, False, True)[0]  # noqa: E731
    x = torch.where(b["mask"], b["lp"], 0.0).double()
    v = torch.where(b["mask"], torch.randn_like(x), 0.0)
    e = 1e-5
    numeric = (f(x + e * v) - f(x - e * v)) / (2 * e)
    # |softplus'''| <= 0.1, along beta times a sum of at most 81 |v|: (0.3 * 81 * 3)^3 e^2 / 6
    assert (numeric - (grad.double() * v).sum()).abs() <= 1e-6 + 2 * R * (grad.double() * v).abs().sum()


@requires_gpu
def test_opcheck_compile_and_layouts():
    b = batch([40, 25], torch.float32, 11, True)
    args = (b["lp"], b["ref"], b["mask"], None, 0.1, "sigmoid", 0.0, 0.0, False, "mean")
    opcheck(preference_loss_fwd, args)
    loss, state = preference_loss_fwd(*args)
    opcheck(preference_loss_bwd, (state, loss, b["mask"], None, list(b["lp"].shape), torch.float32))

    @torch.compile(fullgraph=True)
    def f(lp):
        return preference_loss(lp, b["ref"], b["mask"])

    want, grad = check(b)
    lp = b["lp"].clone().requires_grad_(True)
    got = f(lp)
    got.backward()
    assert torch.equal(got, want) and torch.equal(lp.grad, grad)
    t = lambda x: x.T.contiguous().T  # noqa: E731
    lp = t(b["lp"]).detach().requires_grad_(True)
    got = preference_loss(lp, t(b["ref"]), t(b["mask"]))
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, lp)[0], grad)


@requires_gpu
@pytest.mark.parametrize("lengths", [[300, 5], [9000, 8000]])
def test_captured_and_on_another_stream(lengths):
    b = batch(lengths, torch.float32, 12, False)
    _, grad = check(b)
    lp = b["lp"].clone().requires_grad_(True)
    run = lambda: torch.autograd.grad(preference_loss(lp, b["ref"], b["mask"], b["cu"]), lp)[0]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(run(), grad)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, grad)


@requires_gpu
def test_more_than_2_to_the_31_tokens():
    """Sums of 2^31 equal differences, exact in fp64."""
    T = (1 << 31) + 777
    lp = torch.full((T,), -0.5, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    cu = torch.tensor([0, 1 << 10, T], device="cuda")
    loss, rewards = preference_loss(lp, None, cu_seqlens=cu, beta=1.0, length_normalized=True, return_rewards=True)
    assert rewards.chosen.item() == -0.5 and rewards.rejected.item() == -0.5
    (g,) = torch.autograd.grad(loss, lp)
    assert g[0].item() == -0.5 / 1024 and g[1023] == g[0]
    want = 0.5 / (T - 1024)
    for i in (1024, (1 << 31) - 1, 1 << 31, T - 1):
        assert abs(g[i].item() - want) <= 2.0**-8 * want


@requires_gpu
@pytest.mark.parametrize("smooth", [0.0, 1.0])
def test_impossible_tokens(smooth):
    """A log-probability of -inf in one sequence of a pair: an infinite z, and the sigmoid's term
    of weight 0 is no part of the loss."""
    lp = torch.tensor([[-1.0, -2.0], [-1.5, -0.5], [-1.0, -3.0], [-2.0, -1.0]], device="cuda")
    lp[2 if smooth == 0.0 else 0, 1] = -float("inf")  # z = inf, or -inf where the sign is turned
    lp.requires_grad_(True)
    loss, rewards = preference_loss(lp, beta=0.5, label_smoothing=smooth, reduction="sum", return_rewards=True)
    (grad,) = torch.autograd.grad(loss, lp)
    z = 0.5 * ((-2.0) - (-3.0))  # the second pair, without infinities
    want = math.log1p(math.exp(-z if smooth == 0.0 else z))
    assert abs(loss.item() - want) <= 2.0**-22 * want
    assert (grad[::2] == 0).all()  # the first pair is decided
    slope = 0.5 * (1 / (1 + math.exp(z)) if smooth == 0.0 else 1 / (1 + math.exp(-z)))
    sign = 1.0 if smooth == 0.0 else -1.0
    for row, want in ((1, -sign * slope), (3, sign * slope)):
        assert (grad[row].double() - want).abs().amax() <= 2.0**-22 * slope
    assert rewards.rejected[0].isinf() if smooth == 0.0 else rewards.chosen[0].isinf()
