"""chunked_linear_selective_log_softmax against its definition in 64 bits.

Tolerances (u = 2^-8 for bf16, 2^-11 for fp16, relative):
 * log-probabilities: fp32 logits with the tensor core's accumulation. Each of
   the D / 16 steps may lose up to 2^-23 of the running sum, which is at most
   S = max_v sum_d |H W| / temperature; the target's logit and the log-sum-exp
   each carry that, so |error| <= 2 (D / 16 + 4) 2^-23 S + 2^-20 (exponentials).
 * gradients: each product of a sum carries one rounding of the logits'
   gradient or of e^x (u), in the kept form another of the row (u) and of
   the target's share (u), and the result one of its own (u), or two where
   split-K adds 16-bit halves (2 u). So |error| <= 3 u sum |terms| + 2 u |result|
   plus, where a log-probability is off by e, e p |g| in its term (a
   probability moves by e p, and so does 1 - p at the target).
 * underflow: e^x below 2^-126 counts as 0 (ex2.ftz), and a row stored as e^x
   has a log-sum-exp of at least 2^-64, so a probability may be off by
   2^-126 / 2^-64 = 2^-62 absolutely: 2^-62 |g| sum |H| (or |W|) in the gradients.
   fp16 stores e^x relative to the largest of 128, to a step of 2^-24, and the
   gradient times at least 2^13 / max |g|, to the same step: 2^-25 of a
   probability's largest neighbour and 2^-37 of the largest gradient.
"""

import math

import pytest
import torch
from torch.library import opcheck

from greyhound_b200 import _lib
from greyhound_b200.kernels import linear_logprobs as K
from greyhound_b200.nn.functional import chunked_linear_selective_log_softmax
from greyhound_b200.ops.chunked_linear_selective_log_softmax import (
    linear_selective_log_softmax,
    linear_selective_log_softmax_bwd,
    linear_selective_log_softmax_kept,
    linear_selective_log_softmax_kept_bwd,
)
from greyhound_b200.testing import requires_gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make(N, D, V, dtype, seed, scale=1.0, left_out=0.1, index_dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H = torch.randn(N, D, device="cuda", generator=g).to(dtype)
    W = (torch.randn(V, D, device="cuda", generator=g) * (scale / math.sqrt(D))).to(dtype)
    t = torch.randint(0, V, (N,), device="cuda", generator=g).to(index_dtype)
    if N > 1:
        t[torch.rand(N, device="cuda", generator=g) < left_out] = -100
    return H, W, t, torch.randn(N, device="cuda", generator=g)


def definition(H, W, t, g, temperature=1.0):
    """(logprobs, dH, dW, bounds of the three) in 64 bits."""
    u = U[H.dtype]
    H, W = H.double(), W.double()
    x = H @ W.T / temperature
    lp = torch.log_softmax(x, 1)
    on = t != -100
    at = t.long().clamp(min=0)[:, None]
    y = torch.where(on, lp.gather(1, at)[:, 0], 0.0)
    g = (torch.where(on, g.double(), 0.0) / temperature)[:, None]
    d = torch.zeros_like(x).scatter_(1, at, g) - g * lp.exp()
    S = (H.abs() @ W.abs().T / temperature).amax()
    ey = 2 * (H.shape[1] / 16 + 4) * 2.0**-23 * S + 2.0**-20
    dH, dW = d @ W, d.T @ H
    a = 3 * u * d.abs() + ey * g.abs() * lp.exp()
    bH = a @ W.abs() + 2 * u * dH.abs() + 2.0**-62 * g.abs() * W.abs().sum(0)
    bW = a.T @ H.abs() + 2 * u * dW.abs() + 2.0**-62 * (g.abs() * H.abs()).sum(0)
    if u == 2.0**-11:  # fp16's spacing near zero: of what is stored, and of the results
        V = x.shape[1]
        top = torch.nn.functional.pad(lp.exp(), (0, -V % 128)).view(len(x), -1, 128).amax(2).repeat_interleave(128, 1)[:, :V]
        e = 2.0**-25 * g.abs() * top + 2.0**-37 * g.abs().amax()
        bH, bW = bH + e @ W.abs() + 2.0**-24, bW + e.T @ H.abs() + 2.0**-24
    return y, dH, dW, ey, bH, bW


def check(H, W, t, g, temperature=1.0, **kw):
    h, w = H.clone().requires_grad_(True), W.clone().requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, w, t, temperature=temperature, **kw)
    dh, dw = torch.autograd.grad(y, (h, w), g)
    ry, rH, rW, ey, bH, bW = definition(H, W, t, g, temperature)
    assert y.dtype == torch.float32 and y.shape == t.shape
    assert dh.dtype == H.dtype and dw.dtype == W.dtype
    assert ((y.double() - ry).abs() <= ey).all(), ((y.double() - ry).abs().max(), ey)
    assert ((dh.double() - rH).abs() <= bH).all(), ((dh.double() - rH).abs() / bH).max()
    assert ((dw.double() - rW).abs() <= bW).all(), ((dw.double() - rW).abs() / bW).max()
    skip = t == -100
    assert (y[skip] == 0).all() and (dh[skip] == 0).all()
    return y, dh, dw


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize(
    "N,D,V",
    [(1, 8, 1), (1, 64, 300), (3, 8, 7), (2, 72, 257), (127, 64, 255), (128, 136, 256), (129, 128, 513), (300, 264, 1000),
     (513, 512, 4099), (1030, 320, 2051)],
)
def test_against_definition(N, D, V, dtype):
    check(*make(N, D, V, dtype, N + D + V, scale=2.0))


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("N,D,V", [(1, 512, 1000), (2, 64, 300), (63, 264, 513), (64, 128, 900), (65, 520, 1000), (128, 72, 4099)])
def test_few_rows_round_the_weight_gradient_once(N, D, V, dtype, kept, monkeypatch):
    """Up to 128 rows the second operand of dW's product comes in two parts, u^2 off
    together (plus half of fp16's spacing, 2^-25). The target's term then carries
    that alone, the others two roundings (stored or written, and the row's
    factor), and the result its own u: beside the terms of `definition`
    u |result| + 2 u sum |others| + 2^-14 sum |terms|, with 2^-14 above u^2 and the
    fp32 steps before."""
    if not kept:
        monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    poison = torch.full((1 << 24,), float("nan"), device="cuda")  # what the buffers may find
    del poison
    H, W, t, g = make(N, D, V, dtype, N + D, scale=2.0)
    h, w = H.clone().requires_grad_(True), W.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(chunked_linear_selective_log_softmax(h, w, t), w, g)
    u, (_, _, rW, ey, _, _) = U[dtype], definition(H, W, t, g)
    p = torch.softmax(H.double() @ W.double().T, 1)
    on, at = t != -100, t.clamp(min=0)[:, None]
    ga = torch.where(on, g.double().abs(), 0.0)[:, None]
    others = (ga * p).scatter(1, at, 0.0)
    terms = others.scatter(1, at, ga * (1 - p.gather(1, at)))
    Ha = H.double().abs()
    bound = u * rW.abs() + (2 * u * others + 2.0**-14 * terms + ey * ga * p).T @ Ha + 2.0**-62 * (ga * Ha).sum(0)
    if dtype == torch.float16:
        top = torch.nn.functional.pad(p, (0, -V % 128)).view(N, -1, 128).amax(2).repeat_interleave(128, 1)[:, :V]
        e = 2.0**-25 * ga * top + 2.0**-37 * ga.amax()
        bound += e.T @ Ha + 2.0**-24 * terms.sum(0)[:, None] + 2.0**-24
    assert ((dw.double() - rW).abs() <= bound).all(), ((dw.double() - rW).abs() / bound).max()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("temperature", [0.3, 1.7])
def test_temperature(dtype, temperature):
    check(*make(200, 128, 3001, dtype, 5, scale=1.5), temperature=temperature)


@requires_gpu
@pytest.mark.parametrize("accum", ["fp32", "weight"])
@pytest.mark.parametrize("dtype,keep", [(torch.bfloat16, False), (torch.float16, False), (torch.float16, True)])
def test_backward_over_several_chunks(monkeypatch, dtype, keep, accum):
    """Chunks of 128 rows, the last one short: with fp32 accumulation the same
    bound; in the operand type each of the 4 partial sums is rounded (u each,
    relative to a partial sum of at most the sum of absolute terms)."""
    monkeypatch.setattr(K, "_KEEP_BYTES", K._KEEP_BYTES if keep else 0)
    monkeypatch.setattr(K, "_chunk", lambda N, D, V: 128)
    H, W, t, g = make(400, 128, 1111, dtype, 9, scale=2.0)
    if accum == "fp32":
        check(H, W, t, g)
        return
    h, w = H.clone().requires_grad_(True), W.clone().requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, w, t, grad_weight_accum_dtype=accum)
    _, dw = torch.autograd.grad(y, (h, w), g)
    _, _, rW, _, _, bW = definition(H, W, t, g)
    assert ((dw.double() - rW).abs() <= bW * (7 / 3)).all()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [30.0, 120.0])
def test_logits_outside_the_exponent_window(scale, dtype):
    """Largest logits of about 100 and 400 (e^x as stored in bf16 covers +-44): rows
    are rewritten, with the same bound; p_t near 1 and near 0 both occur."""
    H, W, t, g = make(160, 64, 900, dtype, 3, scale=scale)
    t[::2] = (H[::2].double() @ W.double().T).argmax(1)
    check(H, W, t, g)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_very_small_and_shifted_logits(dtype):
    """Every logit of a row near -400 (below the window), beside normal rows."""
    H, W, t, g = make(130, 64, 700, dtype, 4)
    W[:, 0] = 20.0
    H[:, 0] = 0.0
    H[::3, 0] = -20.0
    H[1::3, 0] = 20.0
    check(H, W, t, g)


@requires_gpu
def test_confident_targets_keep_their_gradient():
    """1 - p_t far below one 16-bit step of p_t."""
    H, W, t, g = make(64, 64, 500, torch.bfloat16, 6, left_out=0.0)
    H[:, 0] = 4.0
    W[:, 0] = 0.0
    W[17, 0] = 4.0
    t[:] = 17
    y, dh, _ = check(H, W, t, g)
    assert (y < 0).all() and (dh != 0).any(1).all()


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept", [True, False])
def test_left_out_rows_may_hold_anything(monkeypatch, kept, dtype):
    if not kept:
        monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    H, W, t, g = make(200, 64, 300, dtype, 8)
    t[5], t[77], t[199] = -100, -100, -100
    clean = check(H, W, t, g)
    H[5], H[77, 3], H[199] = float("nan"), float("inf"), torch.finfo(dtype).max
    g[5], g[77] = float("nan"), float("inf")
    h, w = H.requires_grad_(True), W.requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, w, t)
    dh, dw = torch.autograd.grad(y, (h, w), g)
    assert torch.equal(y.detach(), clean[0].detach()) and torch.equal(dh, clean[1]) and torch.equal(dw, clean[2])


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nan_rows_stay_their_own(dtype):
    H, W, t, g = make(70, 64, 300, dtype, 8, left_out=0.0)
    clean = check(H, W, t, g)
    H[9, 1] = float("nan")
    h = H.requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, W, t)
    (dh,) = torch.autograd.grad(y, h, g)
    rest = torch.arange(70, device="cuda") != 9
    assert y[9].isnan() and dh[9].isnan().all()
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dh[rest], clean[1][rest])


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_gradient_alone_and_no_gradient(dtype):
    H, W, t, g = make(150, 128, 1000, dtype, 11)
    y, dh, dw = check(H, W, t, g)
    assert torch.equal(chunked_linear_selective_log_softmax(H, W, t), y.detach())
    for keep in (K._KEEP_BYTES, 0):
        K._KEEP_BYTES, before = keep, K._KEEP_BYTES
        try:
            h = H.clone().requires_grad_(True)
            (a,) = torch.autograd.grad(chunked_linear_selective_log_softmax(h, W, t), h, g)
            w = W.clone().requires_grad_(True)
            (b,) = torch.autograd.grad(chunked_linear_selective_log_softmax(H, w, t), w, g)
        finally:
            K._KEEP_BYTES = before
        if keep:
            assert torch.equal(a, dh) and torch.equal(b, dw)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1.0, 100.0])
def test_scoring_and_training_forwards_agree_in_every_bit(monkeypatch, scale, dtype):
    """The policy's ratio against log-probabilities taken without a gradient is exactly 1."""
    H, W, t, g = make(300, 192, 1500, dtype, 21, scale=scale)
    scored = chunked_linear_selective_log_softmax(H, W, t)
    h = H.clone().requires_grad_(True)
    assert torch.equal(chunked_linear_selective_log_softmax(h, W, t).detach(), scored)
    monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    assert torch.equal(chunked_linear_selective_log_softmax(h, W, t).detach(), scored)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("D,V", [(8, 1), (8, 9), (264, 3), (72, 257), (1032, 4099), (4096, 20_003), (12_296, 1000), (40_968, 65)])
def test_scoring_few_rows(N, D, V, dtype):
    """One or two rows without a gradient have a kernel of their own, while they fit shared memory."""
    H, W, t, g = make(N, D, V, dtype, N + D, scale=3.0, left_out=0.3)
    for temperature in (1.0, 0.6):
        y = chunked_linear_selective_log_softmax(H, W, t, temperature=temperature)
        ry, _, _, ey, _, _ = definition(H, W, t, g, temperature)
        assert ((y.double() - ry).abs() <= ey).all()
        assert (y[t == -100] == 0).all()


@requires_gpu
def test_scoring_few_rows_with_odd_values():
    H, W, t, g = make(2, 64, 500, torch.bfloat16, 30, left_out=0.0)
    clean = chunked_linear_selective_log_softmax(H, W, t)
    H[1, 5] = float("nan")
    y = chunked_linear_selective_log_softmax(H, W, t)
    assert y[1].isnan() and y[0] == clean[0]
    t[1] = -100
    assert chunked_linear_selective_log_softmax(H, W, t)[1] == 0
    H[1] = 0.0
    W[7, 0] = float("nan")  # one logit of each row
    assert chunked_linear_selective_log_softmax(H, W, t)[0].isnan()


@requires_gpu
def test_retained_graph_takes_other_gradients():
    H, W, t, g = make(150, 128, 1000, torch.bfloat16, 12)
    h, w = H.requires_grad_(True), W.requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, w, t)
    first = torch.autograd.grad(y, (h, w), g, retain_graph=True)
    torch.autograd.grad(y, (h, w), -3 * g, retain_graph=True)
    again = torch.autograd.grad(y, (h, w), g)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@requires_gpu
def test_layouts():
    """Leading dimensions, int32 indices, strided and misaligned operands, an expanded gradient."""
    H, W, t, g = make(120, 64, 333, torch.bfloat16, 13)
    y, dh, dw = check(H, W, t, g)
    y3 = chunked_linear_selective_log_softmax(H.view(4, 30, 64), W, t.view(4, 30).int())
    assert y3.shape == (4, 30) and torch.equal(y3.view(-1), y.detach())
    odd = torch.empty(120 * 64 + 1, dtype=H.dtype, device="cuda")[1:].view(120, 64).copy_(H)
    assert odd.data_ptr() % 16
    wide = torch.empty(333, 128, dtype=W.dtype, device="cuda")[:, ::2].copy_(W)
    assert torch.equal(chunked_linear_selective_log_softmax(odd, wide, t), y.detach())
    h = H.clone().requires_grad_(True)
    chunked_linear_selective_log_softmax(h, W, t).sum().backward()
    ones = torch.autograd.grad(chunked_linear_selective_log_softmax(h, W, t), h, torch.ones(120, device="cuda"))[0]
    assert torch.equal(h.grad, ones)


@requires_gpu
def test_no_rows():
    H = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    W = torch.randn(100, 64, device="cuda").bfloat16().requires_grad_(True)
    y = chunked_linear_selective_log_softmax(H, W, torch.empty(0, device="cuda", dtype=torch.int64))
    dh, dw = torch.autograd.grad(y.sum(), (H, W))
    assert y.shape == (0,) and dh.shape == (0, 64) and (dw == 0).all()


@requires_gpu
def test_bad_index_is_reported_and_harmless():
    H, W, t, g = make(64, 64, 100, torch.bfloat16, 14, left_out=0.0)
    t[3], t[4] = 100, -7
    y = chunked_linear_selective_log_softmax(H, W, t)
    torch.cuda.synchronize()
    assert y[3].isnan() and y[4].isnan() and torch.isfinite(y[5:]).all()
    with pytest.raises(ValueError, match="outside"):
        chunked_linear_selective_log_softmax(H, W, t.clamp(0, 99))


@requires_gpu
def test_against_differences():
    """Directional derivative of the definition, in 64 bits, at two points around H."""
    H, W, t, g = make(48, 64, 200, torch.float16, 15)
    _, dh, _ = check(H, W, t, g)
    v = torch.randn(48, 64, device="cuda", dtype=torch.float64)
    e = 1e-4

    def f(h):
        lp = torch.log_softmax(h @ W.double().T, 1).gather(1, t.clamp(min=0)[:, None])[:, 0]
        return (torch.where(t != -100, lp, 0.0) * g.double()).sum()

    numeric = (f(H.double() + e * v) - f(H.double() - e * v)) / (2 * e)
    # second-order rest of the difference, and the kernel's own bound over the direction
    _, _, _, _, bH, _ = definition(H, W, t, g)
    assert (numeric - (dh.double() * v).sum()).abs() <= (bH * v.abs()).sum() + 1e-4


@requires_gpu
def test_opcheck():
    H, W, t, g = make(40, 64, 130, torch.bfloat16, 16)
    opcheck(linear_selective_log_softmax, (H, W, t, -100, 1.0))
    opcheck(linear_selective_log_softmax_kept, (H, W, t, -100, 1.0), test_utils=["test_schema", "test_faketensor"])
    _, state = linear_selective_log_softmax(H, W, t, -100, 1.0)
    opcheck(linear_selective_log_softmax_bwd, (H, W, t, state, g, -100, 1.0, True, True, False))
    _, kept = linear_selective_log_softmax_kept(H, W, t, -100, 1.0)
    opcheck(linear_selective_log_softmax_kept_bwd, (H, W, kept, g, 1.0, True, True, True))


@requires_gpu
def test_deterministic_and_capturable():
    H, W, t, g = make(300, 128, 2000, torch.bfloat16, 17)
    h, w = H.requires_grad_(True), W.requires_grad_(True)

    def step():
        y = chunked_linear_selective_log_softmax(h, w, t)
        return y, *torch.autograd.grad(y, (h, w), g)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            eager = [a.detach().clone() for a in step()]
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, eager):
        assert torch.equal(a.detach(), b)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_compile(dtype):
    H, W, t, g = make(60, 64, 300, dtype, 18)
    f = torch.compile(chunked_linear_selective_log_softmax, fullgraph=True)
    h, w = H.clone().requires_grad_(True), W.clone().requires_grad_(True)
    y = f(h, w, t, temperature=0.8)
    got = torch.autograd.grad(y, (h, w), g)
    want_y, *want = check(H, W, t, g, temperature=0.8)
    assert torch.equal(y, want_y) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@requires_gpu
@pytest.mark.parametrize("N,V", [(16_300, 131_072), (17_000, 131_072)])
def test_large_products(N, V):
    """N * V beyond 2^31 bytes, kept (4.27 GB of e^x) and, above 4 GiB, recomputed in several
    chunks: some rows of dH and of dW against 64 bits, with the bounds above."""
    H, W, t, g = make(N, 64, V, torch.bfloat16, 19, scale=2.0)
    assert K.keeps_exponentials(H, W) == (N == 16_300)
    h, w = H.requires_grad_(True), W.requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, w, t)
    dh, dw = torch.autograd.grad(y, (h, w), g)
    rows = torch.cat([torch.arange(0, N, 97, device="cuda"), torch.arange(N - 5, N, device="cuda")])
    with torch.no_grad():
        ry, rH, _, ey, bH, _ = definition(H[rows], W, t[rows], g[rows])
        assert ((y[rows].double() - ry).abs() <= ey).all()
        assert ((dh[rows].double() - rH).abs() <= bH).all()
        # columns of the logits' gradient: p from all rows' log-sum-exp
        cols = torch.cat([t[rows[:20]].clamp(min=0), torch.arange(V - 5, V, device="cuda")])
        lse = torch.cat([torch.logsumexp(x.double() @ W.double().T, 1) for x in H.split(1024)])
        x = H.double() @ W[cols].double().T
        gg = torch.where(t != -100, g.double(), 0.0)[:, None]
        p = (x - lse[:, None]).exp()
        d = gg * ((t[:, None] == cols).double() - p)
        u = U[torch.bfloat16]
        rW = d.T @ H.double()
        bW = (3 * u * d.abs() + ey * gg.abs() * p).T @ H.double().abs() + 2 * u * rW.abs()
        assert ((dw[cols].double() - rW).abs() <= bW + 2.0**-62 * (gg.abs() * H.double().abs()).sum(0)).all()


@requires_gpu
def test_scoring_with_trainable_weights_stores_nothing():
    """torch.no_grad with parameters that require a gradient: no e^x is kept (here it would be 200 MB)."""
    H, W, t, _ = make(1000, 64, 100_000, torch.bfloat16, 22)
    w = torch.nn.Parameter(W)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            chunked_linear_selective_log_softmax(H, w, t)
            torch.cuda.synchronize()
            base = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            y = chunked_linear_selective_log_softmax(H, w, t)
            assert torch.cuda.max_memory_allocated() - base < 16 << 20
    assert torch.equal(y, chunked_linear_selective_log_softmax(H, w, t).detach())


@requires_gpu
@pytest.mark.parametrize("kept", [True, False])
def test_result_may_be_changed_in_place(monkeypatch, kept):
    if not kept:
        monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    H, W, t, g = make(50, 64, 300, torch.bfloat16, 23)
    _, dh, _ = check(H, W, t, g)
    h = H.clone().requires_grad_(True)
    y = chunked_linear_selective_log_softmax(h, W, t)
    y.mul_(2.0)
    assert torch.allclose(torch.autograd.grad(y, h, g / 2)[0].float(), dh.float(), rtol=2.0**-7, atol=1e-6)


@requires_gpu
@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("N,D,V", [(3000, 1024, 2048), (1100, 2048, 4096)])
def test_partial_sums_of_the_input_gradient_keep_32_bits(monkeypatch, N, D, V, kept):
    """The two halves of the vocabulary cancel: W is 1 + n in one and -1 + n in the other, p is
    even over both, so that dH = g (W_t - sum p W), with W_t = 0, is small beside its halves of g / 2.
    Some columns of W are random, so that the logits spread by 1/2 and e^x over many 16-bit steps.

    A sum held in 32 bits leaves: the result's rounding u |dH|; the row factor, which takes the
    target's rounding (u at most) off the row's other entries together, u |dH|; the
    log-probability's error ey |dH| likewise; each e^x's own rounding, of at most u and independent:
    by Hoeffding's inequality their sum stays below
    sqrt(2 ln(2 10^13)) u (sum (p W)^2)^(1/2) = 7.9 u (...) for all of 10^7 values but in one draw of
    10^6; and the tensor core's truncation, 2^-23 of the running sum at each of the V / 16 steps.
    16-bit halves would add up to 2^-8 g together."""
    if not kept:
        monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    u = U[torch.bfloat16]
    gen = torch.Generator(device="cuda").manual_seed(35)
    H = torch.zeros(N, D, device="cuda")
    H[:, :64] = torch.randn(N, 64, device="cuda", generator=gen) / 16
    H = H.bfloat16()
    W = torch.randn(V, D, device="cuda", generator=gen) * 0.02
    W[: V // 2] += 1.0
    W[V // 2 :] -= 1.0
    W[:, :64] = torch.randn(V, 64, device="cuda", generator=gen)
    W = W.bfloat16()
    t = torch.randint(0, V, (N,), device="cuda", generator=gen) // 64 * 64
    W[::64] = 0.0
    g = 1.0 + torch.rand(N, device="cuda", generator=gen)
    h = H.clone().requires_grad_(True)
    (dh,) = torch.autograd.grad(chunked_linear_selective_log_softmax(h, W, t), h, g)
    Wd = W.double()
    p = torch.softmax(H.double() @ Wd.T, 1)
    ga = g.double()[:, None]
    want = -ga * (p @ Wd)  # W_t = 0
    S = (H.double().abs() @ Wd.abs().T).amax()
    ey = 2 * (D / 16 + 4) * 2.0**-23 * S + 2.0**-20
    bound = (2 * u + ey) * want.abs() + ga * (7.9 * u * (p**2 @ Wd**2).sqrt() + V / 16 * 2.0**-23 * (p @ Wd.abs()))
    err = (dh.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()

@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("left_out", [None, 0, 1])
def test_scoring_two_rows_in_two_chunks(monkeypatch, dtype, left_out):
    """Each row with its own target, whatever the rows of a chunk."""
    H, W, t, g = make(2, 264, 4099, dtype, 31, scale=3.0, left_out=0.0)
    if left_out is not None:
        t[left_out] = -100
    monkeypatch.setattr(K, "_chunk", lambda N, D, V: 1)
    y = chunked_linear_selective_log_softmax(H, W, t)
    ry, _, _, ey, _, _ = definition(H, W, t, g)
    assert ((y.double() - ry).abs() <= ey).all(), (y, ry)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_c_entry_writes_state_beside_the_kept_buffer(dtype):
    """`state` and `kept` are independent: asking for both gives what each alone does."""
    H, W, t, _ = make(300, 128, 1111, dtype, 32)
    lib = _lib.load()
    N, D, V, code = 300, 128, 1111, _lib.dtype_code(dtype)

    def forward(state, kept):
        out = torch.full((N,), float("nan"), device="cuda")
        ws = _lib.workspace(lib.gh_lsm_fwd_workspace_bytes(N, V, N, int(kept is not None)), H.device)
        st = lib.gh_lsm_fwd(
            H.data_ptr(), W.data_ptr(), t.data_ptr(), _lib.GH_I64, N, D, V, code, -100, 1.0, N, out.data_ptr(),
            _lib.ptr(state), _lib.ptr(kept), 0 if kept is None else kept.numel(), ws.data_ptr(), ws.numel(),
            _lib.stream_handle(H.device),
        )
        _lib.check(st, "forward")
        return out

    alone, both = (torch.full((2, N), float("nan"), device="cuda") for _ in range(2))
    kept = torch.zeros(K.kept_bytes(N, V, dtype), dtype=torch.uint8, device="cuda")
    only = torch.zeros_like(kept)
    y = forward(alone, None)
    assert torch.equal(forward(both, kept), y) and torch.equal(forward(None, only), y)
    assert torch.equal(alone, both) and torch.isfinite(both).all()
    assert torch.equal(kept, only)


@requires_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rest", [100, 300])
def test_chunked_scoring_agrees_with_training_in_every_bit(monkeypatch, dtype, rest):
    """A long chunk and a short last one against the kept forward's single chunk, over
    125 vocabulary tiles: their statistics are added in one order whatever the chunks."""
    H, W, t, _ = make(700 + rest, 192, 32_000, dtype, 33, scale=2.0)
    h = H.clone().requires_grad_(True)
    trained = chunked_linear_selective_log_softmax(h, W, t).detach()
    monkeypatch.setattr(K, "_chunk", lambda N, D, V: 700)
    assert torch.equal(chunked_linear_selective_log_softmax(H, W, t), trained)
    monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    assert torch.equal(chunked_linear_selective_log_softmax(h, W, t).detach(), trained)


@requires_gpu
@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("N", [100, 300])
def test_largest_fp16_hidden_value_with_a_small_gradient(monkeypatch, N, kept):
    """65504 in scored rows whose gradients are 2^-20 to 2^-31 of the largest: the target's entry
    is a subnormal number there, and the row's factor times 65504 must not leave fp16."""
    if not kept:
        monkeypatch.setattr(K, "_KEEP_BYTES", 0)
    H, W, t, g = make(N, 64, 500, torch.float16, 34, left_out=0.0)
    W[:, 3] *= 2.0**-14
    H[::2, 3] = 65504.0
    H[1::4, 3] = -65504.0
    g[1:] = torch.sign(g[1:]) * 2.0 ** -torch.linspace(20, 31, N - 1, device="cuda")
    g[0], H[0, 3] = 1.0, 0.5
    check(H, W, t, g)
