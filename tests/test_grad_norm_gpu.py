"""Global norm and clipping against 64 bits.

Tolerances: squares of fp32 values are summed 8 or 16 at a time in fp32
(17 roundings of 2^-24 at most, on non-negative terms), then in fp64, and the
norm halves the sum's relative error: 2^-20 holds it and the result's rounding.
A clipped element carries the factor's error, the factor's fp32 rounding and
its own product's: 2^-20, plus half a step of its type.
"""

import math

import pytest
import torch

from greyhound_b200.nn.utils import clip_by_global_norm, clip_grad_norm_, global_norm
from greyhound_b200.testing import requires_gpu

E = 2.0**-20
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = list(HALF)


def norm64(ts, kind=2.0):
    flat = torch.cat([t.double().flatten() for t in ts]) if ts else torch.zeros(0, dtype=torch.float64, device="cuda")
    if kind == 2.0:
        return flat.square().sum().sqrt().item()
    return flat.abs().max().item() if flat.numel() else 0.0


def make(shapes, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def check_clip(ts, max_norm, kind=2.0, **kw):
    want = norm64(ts, kind)
    outs, norm = clip_by_global_norm(ts, max_norm, kind, **kw)
    assert abs(norm.item() - want) <= E * want, (norm.item(), want)
    c = min(1.0, max_norm / (want + 1e-6))
    for o, t in zip(outs, ts):
        r = t.double() * c
        tiny = torch.finfo(t.dtype).smallest_normal * HALF[t.dtype] * 2
        assert o.shape == t.shape and o.dtype == t.dtype
        assert ((o.double() - r).abs() <= (E + HALF[t.dtype]) * r.abs() + tiny).all()
    return outs, norm


SHAPES = [
    [(1,)],
    [(7,), (1,), (0,), (31, 3)],
    [(16384,), (16385,), (16383,), (3, 5000), (100_001,)],
    [(513, 257), (513,), (1024, 1024), (0, 4), (2,)] * 8,
]


@requires_gpu
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES], ids=["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: f"{len(s)}x{max(math.prod(x) for x in s)}")
def test_norm_and_clip(shapes, dtypes, kind):
    ts = make(shapes, dtypes, len(shapes))
    assert abs(global_norm(ts, kind).item() - norm64(ts, kind)) <= E * norm64(ts, kind)
    for factor in (0.3, 1.5):
        check_clip(ts, factor * norm64(ts, kind), kind)


@requires_gpu
@pytest.mark.parametrize("count", [96, 97, 288, 289, 896, 897, 2000])
def test_long_lists(count):
    """One launch holds 96, 288 or 896 tensors."""
    ts = make([(i % 40 + 1,) for i in range(count)], TYPES, count)
    check_clip(ts, 0.5 * norm64(ts))
    ref = [t.clone() for t in ts]
    outs, _ = check_clip(ref, 0.5 * norm64(ts))
    clip_by_global_norm(ts, 0.5 * norm64(ref), out=ts)
    assert all(torch.equal(a, b) for a, b in zip(ts, outs))


@requires_gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,to", [(0, 1), (1, 0), (1, 1), (3, 5), (15, 15), (7, 4)])
def test_misaligned_views(dtype, offset, to):
    base = make([(50_020,)], [dtype], 5)[0]
    t = base[offset : offset + 50_001]
    dst = torch.zeros(50_020, dtype=dtype, device="cuda")
    check_clip([t], 0.3 * norm64([t]), out=[dst[to : to + 50_001]])
    assert (dst[:to] == 0).all() and (dst[to + 50_001 :] == 0).all()  # nothing beside the view


@requires_gpu
def test_in_place_and_below_the_limit():
    ts = make([(1000, 7), (33,), (70_000,)], TYPES, 6)
    before = [t.clone() for t in ts]
    outs, norm = clip_by_global_norm(ts, 2 * norm64(ts), out=ts)
    assert all(o.data_ptr() == t.data_ptr() for o, t in zip(outs, ts))
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    want, _ = check_clip(before, 0.1 * norm64(before))
    clip_by_global_norm(ts, 0.1 * norm64(before), out=ts)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))
    mixed = [before[0].clone(), before[1].clone()]
    other = torch.empty_like(mixed[1])
    outs, _ = clip_by_global_norm(mixed, 1e9, out=[mixed[0], other])  # partly in place, below the limit
    assert torch.equal(other, before[1]) and torch.equal(mixed[0], before[0])


@requires_gpu
def test_layouts():
    t = make([(300, 200)], [torch.float32], 7)[0]
    for v in (t.T, t[:, ::2], t[::3], t.view(30, 10, 200).permute(2, 0, 1), t[:1].expand(5, 200)):
        v = v if 0 in v.stride() else v.clone(memory_format=torch.preserve_format) if v.is_contiguous() else v
        check_clip([v], 0.3 * norm64([v]))
    for make_view in (lambda x: x.T, lambda x: x[:, ::2], lambda x: x[1::3]):
        x = t.clone()
        v = make_view(x)
        rest = x.clone()
        want = v.clone()
        clip_by_global_norm([v], 0.3 * norm64([want]), out=[v])
        assert ((v - want * 0.3).abs() <= E * want.abs() + 1e-6 * want.abs()).all()
        make_view(rest).copy_(v)
        assert torch.equal(rest, x)  # the gaps are as they were
    wide = torch.zeros(300, 400, device="cuda")
    check_clip([t], 0.3 * norm64([t]), out=[wide[:, ::2]])
    assert (wide[:, 1::2] == 0).all()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-30, 1e-24, 1e-20, 1e18, 1e25])
def test_squares_beyond_fp32(dtype, size):
    ts = make([(100,), (4000,)], [dtype], 8, scale=size)
    want = norm64(ts)
    assert abs(global_norm(ts).item() - want) <= E * want
    ts.append(torch.zeros(5000, dtype=dtype, device="cuda"))
    assert abs(global_norm(ts).item() - want) <= E * want


@requires_gpu
def test_a_sum_too_long_for_fp32():
    """2^25 ones: an fp32 accumulator would stop at 2^24."""
    t = torch.ones(1 << 25, device="cuda", dtype=torch.bfloat16)
    assert global_norm([t, t]).item() == 2.0**13  # listed twice, counts twice


@requires_gpu
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_nonfinite(kind):
    for bad in (math.nan, math.inf, -math.inf):
        ts = make([(1000,), (20_000,), (3,)], [torch.float32], 9)
        ts[1][777] = bad
        outs, norm = clip_by_global_norm(ts, 1.0, kind)
        assert math.isnan(norm.item()) if math.isnan(bad) else norm.item() == math.inf
        if math.isnan(bad):
            assert all(o.isnan().all() for o in outs)
        else:
            keep = torch.isfinite(ts[1])
            assert (outs[0] == 0).all() and (outs[1][keep] == 0).all() and outs[1][777].isnan()


@requires_gpu
def test_parameters():
    net = torch.nn.Sequential(torch.nn.Linear(60, 33), torch.nn.Linear(33, 9, bias=False)).cuda()
    net[1].weight.requires_grad_(False)
    net(torch.randn(8, 60, device="cuda")).square().sum().backward()
    grads = [p.grad for p in net.parameters() if p.grad is not None]
    before = [g.clone() for g in grads]
    want, n = check_clip(before, 0.25)
    norm = clip_grad_norm_(net.parameters(), 0.25)
    assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(grads, want))
    assert norm.ndim == 0 and norm.dtype == torch.float32 and not norm.requires_grad
    assert clip_grad_norm_(net[1].weight, 1.0).item() == 0.0  # no gradient at all
    one = torch.nn.Parameter(torch.ones(4, device="cuda"))
    one.grad = torch.full((4,), 2.0, device="cuda")
    assert clip_grad_norm_(one, 1e9).item() == 4.0 and (one.grad == 2).all()
    with pytest.raises(ValueError, match="scaled twice"):
        clip_grad_norm_([one, one], 1.0)
    one.grad[1] = math.inf
    with pytest.raises(RuntimeError, match="norm of the gradients"):
        clip_grad_norm_(one, 1.0, error_if_nonfinite=True)
    assert one.grad[0] == 2.0  # not clipped


@requires_gpu
def test_zero_limit_and_zero_gradients():
    ts = make([(100,)], [torch.float32], 10)
    outs, _ = clip_by_global_norm(ts, 0.0)
    assert (outs[0] == 0).all()
    ts[0][3] = math.inf
    outs, norm = clip_by_global_norm(ts, math.inf)
    assert norm.item() == math.inf and torch.equal(outs[0], ts[0])  # no limit, no change
    zero = [torch.zeros(1000, device="cuda")]
    outs, norm = clip_by_global_norm(zero, 1.0)
    assert norm.item() == 0.0 and (outs[0] == 0).all()
    empty = [torch.zeros(0, device="cuda")]
    assert clip_by_global_norm(empty, 1.0)[1].item() == 0.0 and global_norm([]).item() == 0.0


@requires_gpu
def test_overlapping_outputs_are_refused():
    t = torch.ones(100, device="cuda")
    with pytest.raises(ValueError, match="scaled twice"):
        clip_by_global_norm([t[:60], t[40:]], 1.0, out=[t[:60], t[40:]])
    with pytest.raises(ValueError, match="overlaps"):
        clip_by_global_norm([t[:50]], 1.0, out=[t[10:60]])
    assert (t == 1).all()
    assert global_norm([t[:60], t[40:]]).item() == pytest.approx(math.sqrt(120), rel=E)


@requires_gpu
def test_deterministic_and_capturable():
    ts = make([(70_001,), (513, 999), (5,)], TYPES, 11)
    limit = 0.5 * norm64(ts)
    want, n = clip_by_global_norm(ts, limit)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again, n2 = clip_by_global_norm(ts, limit)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(want, again))
    graphs, results = [], []
    for _ in range(2):  # two graphs over the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(clip_by_global_norm(ts, limit))
        graphs.append(graph)
    for graph in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for outs, norm in results:
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(want, outs))


@requires_gpu
def test_more_than_2_to_the_31_elements():
    n = (1 << 31) + 24
    t = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    t[-1], t[1 << 31] = 3.0, 5.0
    want = math.sqrt(n + 8 + 24)
    outs, norm = clip_by_global_norm([t], want / 2, out=[t])
    assert abs(norm.item() - want) <= E * want
    assert outs[0][0] == 0.5 and outs[0][-1] == 1.5 and outs[0][1 << 31] == 2.5
    assert t[(1 << 31) + 1 : -1].eq(0.5).all() and t[: 1 << 20].eq(0.5).all()


@requires_gpu
def test_autograd_notices_clipping_in_place():
    x = torch.randn(1000, device="cuda", requires_grad=True)
    y = x.detach().clone()
    z = (x * y).sum()
    clip_by_global_norm([y], 0.1, out=[y])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        clip_by_global_norm([y.clone()], 0.1, out=[torch.empty_like(y)])


class _Wrapper(torch.Tensor):
    """A tensor without memory of its own, as distributed ones are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        raise NotImplementedError


@requires_gpu
def test_wrappers_around_other_tensors_are_refused():
    t = torch.ones(8, device="cuda")
    with pytest.raises((TypeError, RuntimeError)):
        global_norm([t, _Wrapper(t)])
    with pytest.raises((TypeError, RuntimeError)):
        clip_by_global_norm([_Wrapper(t)], 1.0, out=[t])


@requires_gpu
def test_within_a_compiled_function():
    ts = make([(300,), (17, 9)], TYPES, 12)
    limit = 0.5 * norm64(ts)

    def scaled(a, b):
        (x, y), n = clip_by_global_norm([a + 0.0, b + 0.0], limit)
        return x * 2, y * 2, n

    for got, want in zip(torch.compile(scaled)(*ts), scaled(*ts)):
        assert torch.equal(got, want)


@requires_gpu
def test_outputs_that_overlap_themselves_are_refused_before_anything_is_written():
    a, b = make([(300,), (40, 9)], TYPES[:1], 14)
    wide = torch.ones(1, 7, device="cuda").expand(5, 7)
    keep = [a.clone(), b.clone()]
    for ts, out in (([a, wide, b], None), ([a, b, wide.contiguous()], [a, b, wide]), ([a, b[:, :5], b[:, :5]], None)):
        with pytest.raises(ValueError, match="memory"):
            clip_by_global_norm(ts, 0.1, out=ts if out is None else out)
        assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    # as an input alone it may
    check_clip([a, wide, b], 0.1)


@requires_gpu
def test_compiled_clipping_in_place():
    """Under torch.compile the custom ops change the tensors themselves, and the gradients."""
    ts = make([(300,), (17, 9)], TYPES[:1], 15)
    limit = 0.5 * norm64(ts)

    def in_place(a, b):
        a, b = a * 2.0, b * 2.0
        _, n = clip_by_global_norm([a, b], limit, out=[a, b])
        return a + 1.0, b + 1.0, n

    def gradients(a, b):
        p, q = torch.nn.Parameter(a), torch.nn.Parameter(b)
        (p.square().sum() + q.square().sum()).backward()
        n = clip_grad_norm_([p, q], limit)
        return p.grad, q.grad, n

    for f in (in_place, gradients):
        for got, want in zip(torch.compile(f)(*ts), f(*ts)):
            assert torch.allclose(got, want, rtol=2.0**-22, atol=0.0)
