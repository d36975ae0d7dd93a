"""clipped_policy_loss against its formula in 64 bits.

Tolerances: an fp32 term is e^d from a rounded d, with expf's ulp, a product and
up to three additions of four terms: relative 2^-24 (|d| + 8), of |A| e^d, or of
k (|e^u - 1| + |u|) for the KL term, in which e^u - 1 - u is a difference where
|u| >= 1/2. Further sums are fp64, results fp32 (2^-24) or in the log-probabilities'
type (half a step each).
"""

import math

import pytest
import torch
from _token_batches import HALF, batch
from torch.library import opcheck

from greyhound_b200 import _lib
from greyhound_b200.nn.functional import clipped_policy_loss
from greyhound_b200.ops.token_losses import clipped_policy_loss_bwd, clipped_policy_loss_fwd
from greyhound_b200.testing import requires_gpu

F = 2.0**-24


def reference(lp, old, adv, ref, seq, valid, S, low, high, k, reduction):
    """(loss, its bound, gradient, its bound before the result's rounding, metrics) over flat tokens; ``adv`` per token."""
    lp64, a = lp.double(), adv.double()
    d = lp64 - (lp64 if old is None else old.double())
    r = d.exp()
    clipped = ((a > 0) & (r > 1 + high)) | ((a < 0) & (r < 1 - low))
    l = torch.where(clipped, -r.clamp(1 - low, 1 + high) * a, -r * a)
    g = torch.where(clipped, 0.0, -r * a)
    el = eg = F * (d.abs() + 8) * l.abs()
    kl = torch.zeros_like(l)
    if ref is not None:
        u = ref.double() - lp64
        kl = u.expm1() - u
        el = el + k * F * (u.abs() + 8) * (u.expm1().abs() + u.abs())
        eg = eg + k * F * (u.abs() + 8) * (u.expm1().abs() + g.abs())
        l, g = l + k * kl, g - k * u.expm1()
    n = torch.zeros(S, dtype=torch.float64, device=lp.device).index_add_(0, seq[valid], torch.ones_like(l)[valid])
    if reduction == "sum":
        w = torch.ones_like(l)
    elif reduction == "mean":
        w = torch.full_like(l, 1.0 / max(int(valid.sum()), 1))
    else:
        w = (1.0 / (n.clamp(min=1) * (n > 0).sum().clamp(min=1)))[seq.clamp(min=0)]
    pick = lambda x: torch.where(valid, x * w, 0.0)  # noqa: E731
    loss = pick(l).sum()
    count = max(int(valid.sum()), 1)
    metrics = (kl[valid].sum() / count, clipped[valid].sum() / count, valid.sum())
    return loss, pick(el).sum() + 2 * F * loss.abs(), pick(g), pick(eg) + 4 * F * pick(g).abs(), metrics


def check(b, reduction="mean", k=0.0, per_seq=False, old=True, low=0.2, high=0.3, mask=True, grad_output=1.0, cu32=False):
    adv = b["adv_s"] if per_seq else b["adv"]
    lp = b["lp"].clone().requires_grad_(True)
    cu = b["cu"].int() if cu32 and b["cu"] is not None else b["cu"]
    loss, metrics = clipped_policy_loss(
        lp, b["old"] if old else None, adv, ref_logprobs=b["ref"] if k else None, mask=b["mask"] if mask else None,
        cu_seqlens=cu, clip_low=low, clip_high=high, kl_multiplier=k, reduction=reduction,
        advantages_per="sequence" if per_seq else "token", return_metrics=True)
    (grad,) = torch.autograd.grad(loss, lp, torch.tensor(grad_output, device="cuda"))
    flat = lambda t: t.reshape(-1)  # noqa: E731
    seq = flat(b["seq"])
    valid = flat(b["mask"]) if mask else seq >= 0
    a = b["adv_s"][seq.clamp(min=0)] if per_seq else flat(b["adv"])
    rl, el, rg, eg, rm = reference(
        flat(b["lp"]), flat(b["old"]) if old else None, a, flat(b["ref"]) if k else None, seq, valid, b["S"], low, high, k,
        reduction)
    assert loss.dtype == torch.float32 and loss.ndim == 0 and grad.dtype == b["lp"].dtype and grad.shape == b["lp"].shape
    assert (loss.double() - rl).abs() <= el, (loss, rl, el)
    rg, eg = rg * grad_output, eg * abs(grad_output)
    tiny = torch.finfo(grad.dtype).smallest_normal * HALF[grad.dtype] * 2
    err = (flat(grad).double() - rg).abs()
    assert (err <= eg + HALF[grad.dtype] * rg.abs() + tiny).all(), (err / (eg + HALF[grad.dtype] * rg.abs() + tiny)).max()
    assert (flat(grad)[~valid] == 0).all()
    assert metrics.tokens.item() == rm[2].item()
    assert abs(metrics.clip_fraction.item() - rm[1].item()) <= F
    if k:
        assert abs(metrics.kl.item() - rm[0].item()) <= 2.0**-20 * max(1.0, rm[0].item())
    return loss.detach(), grad


ODD = [[1], [7], [0, 5, 1], [33, 0, 0, 64, 31, 1], [300, 5, 129, 1000], [1] * 40]


@requires_gpu
@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("reduction", ["sum", "mean", "sequence_mean"])
@pytest.mark.parametrize("lengths", ODD, ids=lambda x: f"{len(x)}x{max(x)}")
def test_against_formula(lengths, reduction, padded):
    b = batch(lengths, torch.float32, len(lengths) * 31 + max(lengths), padded, pad=3, front=2, back=5)
    for k in (0.0, 0.1):
        for per_seq in (False, True):
            check(b, reduction, k, per_seq)


@requires_gpu
@pytest.mark.parametrize("reduction", ["sum", "mean", "sequence_mean"])
@pytest.mark.parametrize("lengths", [[9000, 1, 0, 3333], [40] * 700, [100_000, 3], [5, 120_000, 70_001, 0, 2]])
@pytest.mark.parametrize("padded", [True, False])
def test_many_blocks(lengths, reduction, padded):
    if padded and len(lengths) * max(lengths) > 400_000:
        lengths = lengths[:2]
    check(batch(lengths, torch.float32, 3, padded, front=9, back=700), reduction, 0.05, len(lengths) > 3)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("other", [None, torch.float32])
def test_types(dtype, other):
    b = batch([300, 5, 129, 1000], dtype, 4, False, other=other)
    check(b, "mean", 0.1)
    check(b, "sequence_mean", 0.0, grad_output=-2.5, cu32=True)


@requires_gpu
def test_mixed_types_meet_in_fp32():
    b = batch([30, 50], torch.bfloat16, 5, True)
    b["old"] = b["old"].float()
    loss, _ = check(b, "mean", 0.1)
    b["ref"] = b["ref"].float()
    assert torch.equal(check(b, "mean", 0.1)[0], loss)


@requires_gpu
@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("n", [100, 20_000])
def test_nothing_valid(padded, n):
    b = batch([n, 0, 3], torch.float32, 6, padded, left_out=1.1)
    for reduction in ("sum", "mean", "sequence_mean"):
        loss, grad = check(b, reduction, 0.1)
        assert loss == 0 and (grad == 0).all()


@requires_gpu
@pytest.mark.parametrize("shape,cu", [((0,), None), ((0,), [0]), ((0,), [0, 0, 0]), ((0, 5), None), ((5, 0), None), ((4,), [2])])
def test_no_tokens(shape, cu):
    lp = torch.zeros(shape, device="cuda", requires_grad=True)
    c = None if cu is None else torch.tensor(cu, device="cuda", dtype=torch.int32)
    for reduction in ("sum", "mean", "sequence_mean"):
        if cu is None and shape == (0,) or cu is not None or shape:
            loss = clipped_policy_loss(lp, lp.detach(), torch.zeros(shape, device="cuda"), cu_seqlens=c, reduction=reduction,
                                       advantages_per="token")
            (g,) = torch.autograd.grad(loss, lp)
            assert loss == 0 and g.shape == shape and (g == 0).all()


@requires_gpu
def test_on_policy_has_ratio_one():
    b = batch([50, 70], torch.float32, 7, True)
    check(b, "mean", old=False)
    b["old"] = b["lp"].clone()
    check(b, "mean")


@requires_gpu
def test_wide_ratios_and_bounds():
    """Ratios from 0 to inf, advantages of 0, and bounds that never clip."""
    lp = torch.tensor([0.0, -100.0, -1.0, -float("inf"), -3.0, -1.0, -0.1, -50.0], device="cuda")
    old = torch.tensor([-100.0, 0.0, -1.0, -2.0, -200.0, -1.2, -0.1, -0.5], device="cuda")
    adv = torch.tensor([1.0, -1.0, 2.0, -1.0, 1.0, 0.0, 0.0, 1.0], device="cuda")
    b = {"lp": lp, "old": old, "adv": adv, "mask": torch.ones(8, dtype=torch.bool, device="cuda"), "cu": None,
         "seq": torch.zeros(8, dtype=torch.int64, device="cuda"), "S": 1}
    check(b, "sum")
    b = batch([200], torch.float32, 8, False)
    check(b, "mean", low=1.5, high=float("inf"))
    check(b, "mean", low=0.0, high=0.0)


@requires_gpu
def test_side_of_the_border_is_exact():
    """One fp32 step of the log-probability around log(1.2): which side decides whether a token has a gradient."""
    x = torch.tensor(math.log(1.2), dtype=torch.float32).item()
    steps = torch.arange(-8, 9, device="cuda") * 2.0**-26  # an fp32 step near 0.18
    lp = torch.full((17,), x, device="cuda") + steps
    b = {"lp": lp, "old": torch.zeros(17, device="cuda"), "adv": torch.ones(17, device="cuda"), "mask": torch.ones(17, dtype=torch.bool, device="cuda"),
         "cu": None, "seq": torch.zeros(17, dtype=torch.int64, device="cuda"), "S": 1}
    _, g = check(b, "sum", low=0.2, high=0.2)
    assert (g == 0).any() and (g != 0).any()


@requires_gpu
def test_infinite_reference_counts_only_where_it_is_asked_for():
    """ref = inf: the KL term is infinite, and no part of a loss with kl_multiplier 0."""
    lp = torch.tensor([-1.0, -2.0], device="cuda", requires_grad=True)
    ref = torch.tensor([float("inf"), -2.0], device="cuda")
    loss = clipped_policy_loss(lp, None, torch.ones(2, device="cuda"), ref_logprobs=ref)
    assert loss.item() == -1.0 and torch.equal(torch.autograd.grad(loss, lp)[0], torch.full((2,), -0.5, device="cuda"))


@requires_gpu
def test_strides_and_shapes():
    b = batch([40, 25, 3], torch.float32, 9, True)
    loss, grad = check(b, "sequence_mean", 0.1, per_seq=True)
    t = lambda x: x.T.contiguous().T  # noqa: E731
    wide = lambda x: torch.stack([x, x], -1)[..., 0]  # noqa: E731
    for lay in (t, wide):
        lp = lay(b["lp"]).detach().requires_grad_(True)
        other = clipped_policy_loss(lp, lay(b["old"]), b["adv_s"][:, None], lay(b["ref"]), lay(b["mask"]), clip_high=0.3,
                                    kl_multiplier=0.1, reduction="sequence_mean")
        assert torch.equal(other.detach(), loss) and torch.equal(torch.autograd.grad(other, lp)[0], grad)
    expanded = b["adv_s"][:, None].expand(3, 40)
    again = clipped_policy_loss(b["lp"], b["old"], expanded, b["ref"], b["mask"], clip_high=0.3, kl_multiplier=0.1,
                                reduction="sequence_mean")
    assert torch.equal(again, loss)


@requires_gpu
@pytest.mark.parametrize("T", [60, 30_000])
@pytest.mark.parametrize("cu", [[0, 20, 10, 40], [-5, 20, 40, 50], [0, 20, 40, 1 << 40], [50, 40, 30, 0]])
def test_bad_offsets_are_reported(T, cu):
    lp = torch.randn(T, device="cuda", requires_grad=True)
    c = torch.tensor(cu, device="cuda")
    for reduction in ("mean", "sequence_mean"):
        loss = clipped_policy_loss(lp, lp.detach(), torch.ones(3, device="cuda"), cu_seqlens=c, reduction=reduction)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match="offsets"):
            loss.backward()
        loss.backward()  # reported once; nothing faulted
        torch.cuda.synchronize()
        assert _lib.take_device_errors(0) == 0


@requires_gpu
def test_ambiguous_advantages_are_reported():
    lp = torch.randn(3, device="cuda")
    adv = torch.randn(3, device="cuda")
    one = torch.tensor([0, 1, 2, 3], device="cuda")
    assert torch.equal(clipped_policy_loss(lp, None, adv, cu_seqlens=one),
                       clipped_policy_loss(lp, None, adv, cu_seqlens=one, advantages_per="sequence"))
    other = torch.tensor([0, 2, 2, 3], device="cuda")
    clipped_policy_loss(lp, None, adv, cu_seqlens=other)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="advantages_per"):
        clipped_policy_loss(lp, None, adv, cu_seqlens=one)
    for per in ("token", "sequence"):
        clipped_policy_loss(lp, None, adv, cu_seqlens=other, advantages_per=per)
    torch.cuda.synchronize()
    assert _lib.take_device_errors(0) == 0


@requires_gpu
def test_against_differences():
    b = batch([30, 12], torch.float32, 10, True)
    b["adv_s"] *= 0.0
    b["adv_s"] += 1.0
    f = lambda x: reference(x.reshape(-1), b["old"].reshape(-1), torch.ones_like(x.reshape(-1)), b["ref"].reshape(-1),  # noqa: E731
                            b["seq"].reshape(-1), b["mask"].reshape(-1), 2, 0.2, 0.3, 0.1, "sequence_mean")[0]
    _, grad = check(b, "sequence_mean", 0.1, per_seq=True)
    x = b["lp"].double()
    d = (x - b["old"].double())
    near = ((d - math.log(1.3)).abs() < 1e-4) | ((d - math.log(0.8)).abs() < 1e-4)
    v = torch.where(b["mask"] & ~near, torch.randn_like(x), 0.0)
    e = 1e-5
    numeric = (f(x + e * v) - f(x - e * v)) / (2 * e)
    # third derivatives are of the terms' size (< 50 here) and e^2 = 1e-10
    assert (numeric - (grad.double() * v).sum()).abs() <= 1e-7 + 2.0**-20 * (grad.double() * v).abs().sum()


@requires_gpu
def test_opcheck_compile_and_repeat():
    b = batch([40, 25], torch.float32, 11, False)
    args = (b["lp"], b["old"], b["adv"], b["ref"], b["mask"], b["cu"], 0.2, 0.2, 0.1, "mean", "auto", True)
    # the workspace's padding is not written: no comparison of its bytes
    opcheck(clipped_policy_loss_fwd, args, test_utils=["test_schema", "test_faketensor"])
    loss, state = clipped_policy_loss_fwd(*args)
    opcheck(clipped_policy_loss_bwd, (state, b["cu"], loss, list(b["lp"].shape), torch.float32, "mean"))

    @torch.compile(fullgraph=True)
    def f(lp):
        return clipped_policy_loss(lp, b["old"], b["adv"], b["ref"], b["mask"], b["cu"], kl_multiplier=0.1)

    lp = b["lp"].clone().requires_grad_(True)
    got = f(lp)
    got.backward()
    lp2 = b["lp"].clone().requires_grad_(True)
    want = clipped_policy_loss(lp2, b["old"], b["adv"], b["ref"], b["mask"], b["cu"], kl_multiplier=0.1)
    want.backward()
    assert torch.equal(got, want) and torch.equal(lp.grad, lp2.grad)


@requires_gpu
@pytest.mark.parametrize("lengths", [[300, 5], [9000, 8000, 100]])
def test_captured_and_on_another_stream(lengths):
    b = batch(lengths, torch.float32, 12, False)
    loss, grad = check(b, "sequence_mean", 0.1)
    lp = b["lp"].clone().requires_grad_(True)
    run = lambda: torch.autograd.grad(  # noqa: E731
        clipped_policy_loss(lp, b["old"], b["adv"], b["ref"], b["mask"], b["cu"], clip_high=0.3, kl_multiplier=0.1,
                            reduction="sequence_mean"), lp)[0]
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
def test_without_gradients():
    b = batch([300, 5], torch.float32, 13, False)
    loss, _ = check(b, "mean")
    lp = b["lp"].clone().requires_grad_(True)
    with torch.no_grad():
        got = clipped_policy_loss(lp, b["old"], b["adv"], mask=b["mask"], cu_seqlens=b["cu"], clip_high=0.3)
    assert torch.equal(got, loss) and not got.requires_grad


@requires_gpu
def test_more_than_2_to_the_31_tokens():
    """Ratio 1 everywhere: the loss is minus the advantages' mean, weighted by length, and so is the gradient."""
    T = (1 << 31) + 777
    lp = torch.full((T,), -1.0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    cu = torch.tensor([0, 100, (1 << 31) + 5, T - 7], device="cuda")
    adv = torch.tensor([1.0, 2.0, -4.0], device="cuda")
    n = [100, (1 << 31) - 95, 765]
    total = sum(n)
    loss, metrics = clipped_policy_loss(lp, lp.detach(), adv, cu_seqlens=cu, reduction="sum", return_metrics=True)
    want = -(n[0] * 1.0 + n[1] * 2.0 - n[2] * 4.0)
    assert abs(loss.item() - want) <= 2 * F * abs(want)
    assert abs(metrics.tokens.item() - total) <= 2 * F * total
    (g,) = torch.autograd.grad(loss, lp)
    assert g[0] == -1 and g[100] == -2 and g[(1 << 31) + 4] == -2 and g[(1 << 31) + 5] == 4
    mean = clipped_policy_loss(lp, None, torch.full((1,), 3.0, device="cuda"), reduction="sequence_mean")  # one sequence
    assert abs(mean.item() + 3.0) <= 8 * F
    assert abs(torch.autograd.grad(mean, lp)[0][T - 1].item() + 3.0 / T) <= 2.0**-8 * 3.0 / T
    assert g[T - 8] == 4 and (g[T - 7 :] == 0).all() and (g[100 : (1 << 31) + 5 : 4099] == -2).all()


@requires_gpu
@pytest.mark.parametrize("reduction", ["sum", "mean", "sequence_mean"])
@pytest.mark.parametrize("T", [5, 20_000])
def test_no_sequences(T, reduction):
    """Offsets of no sequence: no token counts, and per-sequence advantages are empty."""
    lp = torch.full((T,), float("nan"), device="cuda", requires_grad=True)
    cu = torch.tensor([3], device="cuda")
    for adv in (torch.empty(0, device="cuda"), torch.ones(T, device="cuda")):
        loss, metrics = clipped_policy_loss(lp, None, adv, cu_seqlens=cu, reduction=reduction, return_metrics=True)
        (grad,) = torch.autograd.grad(loss, lp)
        assert loss == 0 and metrics.tokens == 0 and (grad == 0).all()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ratio_is_one_without_old_logprobs(dtype):
    """Also for a token of log-probability -inf; a NaN stays one."""
    lp = torch.tensor([-1.0, -float("inf"), -3.0, 0.0], device="cuda", dtype=dtype, requires_grad=True)
    adv = torch.tensor([1.0, -2.0, 0.5, 4.0], device="cuda")
    loss = clipped_policy_loss(lp, None, adv, reduction="sum")
    (grad,) = torch.autograd.grad(loss, lp)
    assert loss == -3.5 and torch.equal(grad.float(), -adv)
    lp = torch.tensor([-1.0, float("nan")], device="cuda", dtype=dtype)
    assert clipped_policy_loss(lp, None, adv[:2]).isnan()
