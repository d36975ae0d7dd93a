"""The operators run together, as a training step chains them: log-probabilities from
hidden states, a loss over them, the backward through both, and clipping.

Against the same chain in 64 bits. The log-probabilities' bound e (see
test_linear_logprobs_gpu) moves a ratio by a factor e^e and a preference margin by
beta e per token; 2^-8 relative to the gradients' largest entries, the 16-bit
operands' step, is far above both at these sizes, and the three roundings of
the products behind it (1.2 %) are what the comparison allows: 2^-6 of the largest.
"""

import math

import pytest
import torch

from greyhound_b200 import _lib
from greyhound_b200.nn.functional import (
    chunked_linear_selective_log_softmax,
    clipped_policy_loss,
    preference_loss,
    selective_log_softmax,
)
from greyhound_b200.nn.utils import clip_grad_norm_
from greyhound_b200.testing import requires_gpu


def model(seed=0, tokens=230, hidden=128, vocab=1500):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, device="cuda", generator=g).bfloat16()
    body = (torch.eye(hidden, device="cuda") + 0.1 * torch.randn(hidden, hidden, device="cuda", generator=g)).bfloat16()
    head = (torch.randn(vocab, hidden, device="cuda", generator=g) * 0.1).bfloat16()
    index = torch.randint(0, vocab, (tokens,), device="cuda", generator=g)
    return x, body, head, index, g


def reference_logprobs(x, body, head, index, temperature=1.0):
    h = (x.double() @ body.double().T)
    return torch.log_softmax(h @ head.double().T / temperature, 1).gather(1, index.clamp(min=0)[:, None])[:, 0]


def compare(grads, ref, tol=2.0**-6):
    for a, b in zip(grads, ref):
        assert (a.double() - b).abs().max() <= tol * b.abs().max(), ((a.double() - b).abs().max() / b.abs().max())


@requires_gpu
@pytest.mark.parametrize("reduction", ["mean", "sequence_mean"])
def test_policy_step(reduction):
    x, body, head, index, g = model(1)
    cu = torch.tensor([0, 40, 40, 150, 220], device="cuda", dtype=torch.int32)
    index[:5] = -100  # a prompt, and ten tokens behind the last sequence
    mask = index != -100
    with torch.no_grad():
        old = chunked_linear_selective_log_softmax(x @ body.T, head, index, temperature=0.8)
        ref = chunked_linear_selective_log_softmax(x, head, index, temperature=0.8)
    adv = torch.randn(4, device="cuda", generator=g)
    params = [torch.nn.Parameter((body + 0.02 * torch.randn_like(body))), torch.nn.Parameter(head.clone())]
    lp = chunked_linear_selective_log_softmax(x @ params[0].T, params[1], index, temperature=0.8)
    loss, metrics = clipped_policy_loss(lp, old, adv, ref, mask, cu, kl_multiplier=0.1, reduction=reduction,
                                        advantages_per="sequence", return_metrics=True)
    loss.backward()
    # the chain in 64 bits from the same hidden states, whose product is torch's own
    h = (x @ params[0].detach().T).double().requires_grad_(True)
    w = params[1].detach().double().requires_grad_(True)
    l64 = torch.log_softmax(h @ w.T / 0.8, 1).gather(1, index.clamp(min=0)[:, None])[:, 0]
    seq = torch.bucketize(torch.arange(230, device="cuda"), cu.long(), right=True) - 1
    ok = mask & (seq < 4)
    seq = seq.clamp(max=3)
    r = torch.exp(l64 - old.double())
    a = adv.double()[seq]
    u = ref.double() - l64
    term = torch.where(ok, -torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.1 * (u.exp() - u - 1), 0.0)
    n = torch.zeros(4, dtype=torch.float64, device="cuda").index_add(0, seq, ok.double())
    want = term.sum() / ok.sum() if reduction == "mean" else (term / n.clamp(min=1)[seq]).sum() / (n > 0).sum()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-4 * term.abs().max().item()
    assert metrics.tokens.item() == ok.sum().item()
    compare([params[0].grad, params[1].grad], [h.grad.T @ x.double(), w.grad])
    before = [p.grad.clone() for p in params]
    total = math.sqrt(sum(b.double().square().sum().item() for b in before))
    norm = clip_grad_norm_(params, 0.5 * total)
    assert norm.item() == pytest.approx(total, rel=1e-5)
    for p, b in zip(params, before):
        assert (p.grad.double() - 0.5 * b.double()).abs().max() <= 2.0**-8 * b.abs().max()


@requires_gpu
def test_on_policy_ratio_is_exactly_one():
    """Scoring and training passes over the same rows: no token is clipped by rounding, with bounds of 0."""
    x, body, head, index, g = model(2)
    adv = torch.randn(230, device="cuda", generator=g)
    h = (x @ body.T).requires_grad_(True)
    with torch.no_grad():
        old = chunked_linear_selective_log_softmax(h, head, index)
    lp = chunked_linear_selective_log_softmax(h, head, index)
    loss, metrics = clipped_policy_loss(lp, old, adv, clip_low=0.0, clip_high=0.0, return_metrics=True)
    assert metrics.clip_fraction.item() == 0.0
    assert loss.item() == pytest.approx(-adv.double().mean().item(), rel=1e-6, abs=1e-8)
    none = clipped_policy_loss(lp, None, adv)
    assert torch.equal(none, loss)


@requires_gpu
@pytest.mark.parametrize("linear", [True, False])
def test_preference_step(linear):
    """From hidden states, and from materialised logits through selective_log_softmax."""
    x, body, head, index, g = model(3, tokens=4 * 50)
    mask = (torch.arange(50, device="cuda") < torch.tensor([50, 33, 1, 48], device="cuda")[:, None])
    index = torch.where(mask.view(-1), index, 0)
    ref = reference_logprobs(x, body, head, index).float().view(4, 50)
    head = (head + 0.02 * torch.randn_like(head)).requires_grad_(True)
    h = (x @ body.T).requires_grad_(True)
    if linear:
        lp = chunked_linear_selective_log_softmax(h.view(4, 50, -1), head, torch.where(mask, index.view(4, 50), -100))
    else:
        lp = selective_log_softmax((h.float() @ head.float().T).view(4, 50, -1), index.view(4, 50))
    loss, rewards = preference_loss(lp, ref, mask, beta=0.3, return_rewards=True)
    loss.backward()
    h64, w64 = h.detach().double().requires_grad_(True), head.detach().double().requires_grad_(True)
    l64 = torch.log_softmax(h64 @ w64.T, 1).gather(1, index[:, None])[:, 0].view(4, 50)
    s = torch.where(mask, l64 - ref.double(), 0.0).sum(1)
    want = -torch.nn.functional.logsigmoid(0.3 * (s[:2] - s[2:])).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    assert torch.allclose(torch.cat([rewards.chosen, rewards.rejected]).double(), 0.3 * s.detach(), atol=1e-4)
    compare([h.grad, head.grad], [h64.grad, w64.grad])
    assert (h.grad.view(4, 50, -1)[~mask] == 0).all()


@requires_gpu
def test_captured_policy_step():
    """The whole step in one graph, twice, with new inputs copied in between."""
    x, body, head, index, g = model(4)
    adv = torch.randn(230, device="cuda", generator=g)
    h = (x @ body.T).requires_grad_(True)
    w = head.requires_grad_(True)

    def step():
        lp = chunked_linear_selective_log_softmax(h, w, index)
        loss = clipped_policy_loss(lp, old, adv, clip_high=0.3)
        grads = torch.autograd.grad(loss, (h, w))
        return loss, *grads

    from greyhound_b200.nn.utils import clip_by_global_norm

    with torch.no_grad():
        old = chunked_linear_selective_log_softmax(h, w, index) + 0.3 * torch.randn(230, device="cuda", generator=g)

    def full():
        loss, *grads = step()
        clipped, norm = clip_by_global_norm(grads, 1e-3)
        return loss, norm, *clipped

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = [a.detach().clone() for a in full()]
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = full()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, first))
    adv.neg_()
    graph.replay()
    other = full()
    assert all(torch.equal(a, b) for a, b in zip(out, other)) and not torch.equal(out[0], first[0])
    torch.cuda.synchronize()
    assert _lib.take_device_errors(0) == 0
