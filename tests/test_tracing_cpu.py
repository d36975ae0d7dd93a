"""What a trace records of the log-probabilities, the token losses and the clipping: their
custom ops, forward and backward. The kernels' wrappers are replaced by ones that write
past the dispatcher, as the C entries do."""

import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from greyhound_b200.nn import utils
from greyhound_b200.nn.functional import chunked_linear_selective_log_softmax, clipped_policy_loss, preference_loss
from greyhound_b200.ops import chunked_linear_selective_log_softmax as lsm
from greyhound_b200.ops import grad_norm, token_losses


def written(*shape, dtype=torch.float32):
    """A tensor whose contents no dispatcher sees being written."""
    t = torch.empty(shape, dtype=dtype)
    flat = torch.full(shape, 7.0, dtype=dtype)
    ctypes.memmove(t.data_ptr(), flat.data_ptr(), t.numel() * t.element_size())
    return t


@pytest.fixture
def kernels(monkeypatch):
    def policy(logprobs, *a):
        return written(), written(4 + logprobs.numel())

    monkeypatch.setattr(token_losses, "policy_loss_forward", policy)
    monkeypatch.setattr(token_losses, "policy_state_size", lambda lp, *a: 4 + lp.numel())
    monkeypatch.setattr(token_losses, "policy_loss_backward", lambda st, cu, g, shape, dt, red: written(*shape, dtype=dt))
    monkeypatch.setattr(token_losses, "preference_loss_forward", lambda lp, *a: (written(), written(2, lp.shape[0])))
    monkeypatch.setattr(
        token_losses, "preference_loss_backward", lambda st, g, m, cu, shape, dt: written(*shape, dtype=dt)
    )

    def linear(h, w, t, ignore, temperature, want_state=False, keep=False):
        return written(len(h)), written(2, len(h)) if want_state else None, written(8, dtype=torch.uint8) if keep else None

    monkeypatch.setattr(lsm, "linear_logprobs", linear)
    monkeypatch.setattr(lsm, "kept_bytes", lambda *a: 8)
    monkeypatch.setattr(lsm, "linear_logprobs_backward_kept", lambda h, w, *a: (written(*h.shape), written(*w.shape)))
    monkeypatch.setattr(lsm, "linear_logprobs_backward", lambda h, w, *a: (written(*h.shape), written(*w.shape)))


def head(x):  # weight and index, made of the input for the fake mode's sake
    return x.detach().repeat(2, 1), x.detach()[:, 0].long()


def policy_step(x):
    loss = clipped_policy_loss(x, None, torch.ones_like(x))
    return loss, torch.autograd.grad(loss, x)[0]


def preference_step(x):
    loss = preference_loss(x)
    return loss, torch.autograd.grad(loss, x)[0]


def linear_step(x):
    y = chunked_linear_selective_log_softmax(x, *head(x))
    return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]


def scoring(x):
    return chunked_linear_selective_log_softmax(x.detach(), *head(x)), x * 7.0


STEPS = [
    (policy_step, (4, 2), {"clipped_policy_loss_fwd", "clipped_policy_loss_bwd"}),
    (preference_step, (4, 2), {"preference_loss_fwd", "preference_loss_bwd"}),
    (linear_step, (4, 8), {"linear_selective_log_softmax_kept", "linear_selective_log_softmax_kept_bwd"}),
    (scoring, (4, 8), {"linear_selective_log_softmax"}),
]


class Recorder(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "greyhound":
            self.ops.add(func._opname)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("step,shape,ops", STEPS)
def test_make_fx_records_the_ops(kernels, step, shape, ops, mode):
    x = torch.ones(*shape, requires_grad=True)
    graph = make_fx(step, tracing_mode=mode)(x)
    assert {n.target._opname for n in graph.graph.nodes if getattr(n.target, "namespace", "") == "greyhound"} == ops
    for _ in range(3):
        for got, want in zip(graph(x), step(x)):
            assert torch.equal(got, want) and (want == 7.0).all()


@pytest.mark.parametrize("step,shape,ops", STEPS)
def test_dispatch_modes_see_the_ops(kernels, step, shape, ops):
    with Recorder() as seen:
        step(torch.ones(*shape, requires_grad=True))
    assert seen.ops == ops


@pytest.mark.parametrize("step,shape,ops", STEPS)
def test_outside_of_tracing_no_op_is_called(kernels, step, shape, ops, monkeypatch):
    for name in ops:
        module = token_losses if "loss" in name else lsm
        monkeypatch.setattr(module, name, None)
    assert (step(torch.ones(*shape, requires_grad=True))[0] == 7.0).all()


@pytest.fixture
def clipping(monkeypatch):
    def tensors(ts, outs, max_norm, kind, device):
        for t, o in zip(ts, outs or ()):
            half = t.detach() * 0.5
            ctypes.memmove(o.data_ptr(), half.data_ptr(), o.numel() * 4)
            torch.autograd.graph.increment_version(o)
        return written()

    monkeypatch.setattr(grad_norm, "clip_tensors", tensors)


def norm_alone(a, b):
    return (utils.global_norm([a, b]),)


def clipped_copies(a, b):
    (x, y), n = utils.clip_by_global_norm([a, b], 1.0)
    return x + 1.0, y + 1.0, n


def clipped_in_place(a, b):
    ts = [a + 1.0, b + 1.0]
    _, n = utils.clip_by_global_norm(ts, 1.0, out=ts)
    return ts[0] * 3.0, ts[1] * 3.0, n


def one_in_place(a, b):
    a, b, c = a + 1.0, b + 1.0, torch.empty_like(b)
    _, n = utils.clip_by_global_norm([a, b], 1.0, out=[a, c])
    return a * 3.0, b * 3.0, c * 3.0, n


def parameters(a, b):
    p, q = torch.nn.Parameter(a + 1.0), torch.nn.Parameter(b + 1.0)
    p.grad, q.grad = a + 2.0, b + 3.0
    n = utils.clip_grad_norm_([p, q], 1.0)
    return p.grad * 3.0, q.grad * 3.0, n


CLIPS = [
    (norm_alone, {"global_norm"}),
    (clipped_copies, {"clip_by_global_norm_out"}),
    (clipped_in_place, {"clip_by_global_norm_"}),
    (one_in_place, {"clip_by_global_norm_out"}),
    (parameters, {"clip_by_global_norm_"}),
]


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("step,ops", CLIPS)
def test_make_fx_records_the_clipping(clipping, step, ops, mode):
    a, b = torch.randn(3), torch.randn(2, 5)
    graph = make_fx(step, tracing_mode=mode)(a, b)
    assert {n.target._opname for n in graph.graph.nodes if getattr(n.target, "namespace", "") == "greyhound"} == ops
    for _ in range(2):
        for got, want in zip(graph(a, b), step(a, b)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("step,ops", CLIPS)
def test_dispatch_modes_see_the_clipping(clipping, step, ops):
    with Recorder() as seen:
        step(torch.randn(3), torch.randn(2, 5))
    assert seen.ops == ops


@pytest.mark.parametrize("step", [s for s, _ in CLIPS if s is not parameters])
def test_jit_traces_hold_the_clipping(clipping, step):
    a, b = torch.randn(3), torch.randn(2, 5)
    graph = torch.jit.trace(step, (a, b), check_trace=False)
    a, b = torch.randn(3), torch.randn(2, 5)
    for got, want in zip(graph(a, b), step(a, b)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("step", [s for s, _ in CLIPS if s is not parameters])
def test_compiled_clipping(clipping, step):
    a, b = torch.randn(3), torch.randn(2, 5)
    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    for got, want in zip(compiled(a, b), step(a, b)):
        assert torch.equal(got, want)
