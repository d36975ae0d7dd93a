"""Workloads of the reinforcement- and preference-training operators.

Four operators, as one training step chains them: log-probabilities of given
tokens from hidden states and the head's weight (``linear_logprobs``), the
clipped policy loss (``policy``) and the paired preference loss
(``preference``) over such log-probabilities, and the global gradient norm with
clipping (``clip``). ``run`` computes them in a plain form, or, with ``own``
set, through greyhound_b200.
"""

import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------
# Cases


def listed():
    return [
        # One new token scored against the full vocabulary: reading the weight once is all there is.
        {"name": "logprobs_one_token", "op": "linear_logprobs", "rows": 1, "hidden": 4096, "vocab": 128256, "dtype": "bf16",
         "temperature": 1.0, "train": False},
        # A small model's training step, both gradients.
        {"name": "logprobs_train_512", "op": "linear_logprobs", "rows": 512, "hidden": 1024, "vocab": 32000, "dtype": "bf16",
         "temperature": 1.0, "train": True},
        # Half precision, sampled at a temperature, with no size a multiple of a tile.
        {"name": "logprobs_train_ragged_fp16", "op": "linear_logprobs", "rows": 777, "hidden": 1000, "vocab": 32003,
         "dtype": "fp16", "temperature": 0.7, "train": True},
        # The benchmark's head at its own size: forward and both gradients.
        {"name": "logprobs_train_8192", "op": "linear_logprobs", "rows": 8192, "hidden": 4096, "vocab": 128256, "dtype": "bf16",
         "temperature": 1.0, "train": True},
        # A micro-batch of packed answers: a few thousand tokens, where latency counts.
        {"name": "policy_few_tokens", "op": "policy", "seqs": 16, "longest": 400, "packed": True, "dtype": "fp32",
         "per_token": False, "kl": 0.0, "reduction": "mean"},
        # A whole rollout batch, padded, with a mask, the KL term and one advantage an answer.
        {"name": "policy_padded_batch", "op": "policy", "seqs": 512, "longest": 4096, "packed": False, "dtype": "fp32",
         "per_token": False, "kl": 0.05, "reduction": "mean"},
        # Packed answers, every answer weighing the same, log-probabilities in the logits' 16 bits.
        {"name": "policy_packed_sequence_mean", "op": "policy", "seqs": 96, "longest": 5001, "packed": True, "dtype": "bf16",
         "per_token": True, "kl": 0.02, "reduction": "sequence_mean"},
        # A micro-batch of preference pairs.
        {"name": "preference_few_pairs", "op": "preference", "pairs": 8, "longest": 300, "packed": True, "dtype": "fp32",
         "kind": "sigmoid", "smoothing": 0.0, "normalized": False},
        # A large batch of long pairs, padded, with smoothed labels and sums weighted by length.
        {"name": "preference_long_pairs", "op": "preference", "pairs": 128, "longest": 8192, "packed": False, "dtype": "fp32",
         "kind": "sigmoid", "smoothing": 0.1, "normalized": True},
        # A small model's many small gradients (vectors, odd matrices), over the limit: norm and scaling.
        {"name": "clip_many_small", "op": "clip", "layers": 24, "hidden": 513, "vocab": 0, "dtype": "bf16", "in_place": False},
        # Gradients below the limit, clipped in place: the norm is read, nothing changes.
        {"name": "clip_below_limit", "op": "clip", "layers": 16, "hidden": 2048, "vocab": 0, "dtype": "fp32", "in_place": True},
        # The benchmark's head gradient with some layers' behind it, over the limit.
        {"name": "clip_head_and_layers", "op": "clip", "layers": 4, "hidden": 4096, "vocab": 128256, "dtype": "bf16",
         "in_place": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear_logprobs", "policy", "preference", "clip"])
    if op == "linear_logprobs":
        hidden, vocab = 8 * _log(rng, 8, 512), _log(rng, 1000, 128256)
        most = 8192 * 4096 * 128256 // (hidden * vocab)
        return {"op": op, "rows": min(_log(rng, 1, 20000), most, (1 << 31) // vocab), "hidden": hidden, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]),
                "train": rng.random() < 0.7}
    if op == "policy":
        longest = _log(rng, 1, 8192)
        return {"op": op, "seqs": _log(rng, 1, max(2, min(512, (1 << 21) // longest))), "longest": longest,
                "packed": rng.random() < 0.5, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "per_token": rng.random() < 0.5, "kl": rng.choice([0.0, 0.01, 0.1]),
                "reduction": rng.choice(["mean", "sum", "sequence_mean"])}
    if op == "preference":
        longest = _log(rng, 1, 8192)
        return {"op": op, "pairs": _log(rng, 1, max(2, min(256, (1 << 20) // longest))), "longest": longest,
                "packed": rng.random() < 0.5, "dtype": rng.choice(["fp32", "fp32", "bf16"]),
                "kind": rng.choice(["sigmoid", "hinge", "ipo"]), "smoothing": rng.choice([0.0, 0.1]),
                "normalized": rng.random() < 0.5}
    return {"op": op, "layers": _log(rng, 1, 24), "hidden": _log(rng, 16, 2048), "vocab": _log(rng, 1000, 128256),
            "dtype": rng.choice(["bf16", "fp32", "fp16"]), "in_place": rng.random() < 0.4}


def _lengths(count, longest, seed):
    """Answer lengths of one batch: one of the longest, one that is empty, the rest between. The seed sets their order, not their sum."""
    rng = random.Random(count * 8209 + longest)
    lengths = [rng.randint(max(1, longest // 8), longest) for _ in range(count)]
    lengths[0] = longest
    if count > 2:
        lengths[1] = 0
    random.Random(seed).shuffle(lengths)
    return lengths


def _shapes(case):
    """Gradients of a small decoder: per layer four matrices and two vectors, and the head's."""
    h = case["hidden"]
    per = [(h, h), (h, 4 * h), (4 * h, h), (h, max(1, h // 4)), (h,), (h,)]
    return per * case["layers"] + ([(case["vocab"], h)] if case["vocab"] else [])


# --------------------------------------------------------------------------
# What a program has in hand


def _tokens(case, seed):
    """Log-probabilities under the policy, the sampling policy and the reference, padded or packed."""
    count = case["seqs"] if case["op"] == "policy" else 2 * case["pairs"]
    lengths = _lengths(count, case["longest"], seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n = torch.tensor(lengths, device="cuda")
    if case["packed"]:
        shape, mask = (sum(lengths),), None
        cu = torch.zeros(count + 1, dtype=torch.int32, device="cuda")
        cu[1:] = n.cumsum(0)
    else:
        shape, cu = (count, case["longest"]), None
        mask = torch.arange(case["longest"], device="cuda") < n[:, None]

    def normal(*size):
        return torch.randn(size, generator=gen, device="cuda")

    dtype = DTYPES[case["dtype"]]
    logprobs = (-normal(*shape).abs() * 1.5).to(dtype)
    old = (logprobs.float() + 0.15 * normal(*shape)).to(dtype)
    ref = (logprobs.float() + 0.3 * normal(*shape)).to(dtype)
    per_token = case["op"] == "policy" and case["per_token"]
    advantages = normal(*(shape if per_token else (count,)))
    return {"logprobs": logprobs.requires_grad_(True), "old": old, "ref": ref, "advantages": advantages, "mask": mask, "cu": cu}


def _buckets(case, dtype):
    """One flat buffer and the gradients as views of it, each on a boundary of eight values, as a data-parallel program keeps them."""
    shapes = _shapes(case)
    slots = [-(-math.prod(s) // 8) * 8 for s in shapes]
    flat = torch.zeros(sum(slots), dtype=dtype, device="cuda")
    return flat, [piece[: math.prod(s)].view(s) for piece, s in zip(flat.split(slots), shapes)]


def prepare(case, seed):
    state = {"case": dict(case)}
    if case["op"] in ("policy", "preference"):
        state.update(_tokens(case, seed))
        return state
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "clip":
        flat, grads = _buckets(case, dtype)
        for g in grads:
            g.copy_(0.02 * torch.randn(g.shape, generator=gen, device="cuda"))
        # 0.02 * sqrt(elements) is the norm to be expected
        norm = 0.02 * math.sqrt(sum(g.numel() for g in grads))
        state.update(grads=grads, max_norm=2.0 * norm if case["in_place"] else 0.3 * norm)
        state["flat"], state["out"] = (flat, grads) if case["in_place"] else _buckets(case, dtype)
        return state
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    inputs = torch.randn((rows, hidden), generator=gen, device="cuda").to(dtype)
    weight = (torch.randn((vocab, hidden), generator=gen, device="cuda") * 0.02).to(dtype)  # the benchmark's distributions
    index = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    if rows > 1:  # prompt and padding rows: not scored
        index[torch.rand(rows, generator=gen, device="cuda") < 0.02] = IGNORE
    grad = torch.randn(rows, generator=gen, device="cuda") / rows
    state.update(inputs=inputs.requires_grad_(case["train"]), weight=weight.requires_grad_(case["train"]), index=index, grad=grad)
    return state


# --------------------------------------------------------------------------
# One pass


def _linear_logprobs(s):
    c = s["case"]
    if own:
        from greyhound_b200.nn.functional import chunked_linear_selective_log_softmax

        logprobs = chunked_linear_selective_log_softmax(s["inputs"], s["weight"], s["index"], temperature=c["temperature"])
        if not c["train"]:
            return logprobs
        return [logprobs.detach(), *torch.autograd.grad(logprobs, (s["inputs"], s["weight"]), s["grad"])]
    h, w, index = s["inputs"].detach().float(), s["weight"].detach().float(), s["index"]
    logits = (h @ w.T) / c["temperature"]
    scored = index != IGNORE
    target = torch.where(scored, index, 0)[:, None]
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    logprobs = torch.where(scored, (logits.gather(1, target) - lse)[:, 0], 0.0)
    if not c["train"]:
        return logprobs
    g = torch.where(scored, s["grad"], 0.0)[:, None] / c["temperature"]
    d = (logits - lse).exp() * -g
    d.scatter_add_(1, target, g)
    return [logprobs, (d @ w).to(s["inputs"].dtype), (d.T @ h).to(s["weight"].dtype)]


def _token_rows(s):
    """(sequence of each token, which tokens count, tokens of each sequence) of a padded or packed batch."""
    lp = s["logprobs"]
    if s["cu"] is None:
        count, length = lp.shape
        seq = torch.arange(count, device=lp.device)[:, None].expand(count, length)
        return seq, s["mask"], s["mask"].sum(1)
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    return torch.repeat_interleave(torch.arange(len(n), device=lp.device), n, output_size=lp.numel()), torch.ones_like(lp, dtype=torch.bool), n


def _policy(s):
    c = s["case"]
    if own:
        from greyhound_b200.nn.functional import clipped_policy_loss

        loss = clipped_policy_loss(s["logprobs"], s["old"], s["advantages"], ref_logprobs=s["ref"] if c["kl"] else None,
                                   mask=s["mask"], cu_seqlens=s["cu"], clip_low=0.2, clip_high=0.28, kl_multiplier=c["kl"],
                                   reduction=c["reduction"])
        return [loss.detach(), *torch.autograd.grad(loss, s["logprobs"])]
    seq, valid, n = _token_rows(s)
    # 64 bits: which side of a clip border a token is on, and long sums
    lp = s["logprobs"].detach().double()
    a = s["advantages"].double()
    a = a if c["per_token"] else a[seq]
    r = (lp - s["old"].double()).exp()
    clipped = ((a > 0) & (r > 1.28)) | ((a < 0) & (r < 0.8))
    loss = torch.where(clipped, -r.clamp(0.8, 1.28) * a, -r * a)
    d = torch.where(clipped, 0.0, -r * a)
    if c["kl"]:
        u = s["ref"].double() - lp
        loss = loss + c["kl"] * (u.expm1() - u)
        d = d - c["kl"] * u.expm1()
    if c["reduction"] == "sum":
        weight = torch.ones_like(loss)
    elif c["reduction"] == "mean":
        weight = 1.0 / valid.sum().clamp(min=1).double()
    else:
        weight = (1.0 / (n.clamp(min=1) * (n > 0).sum().clamp(min=1)).double())[seq]
    loss, d = torch.where(valid, loss * weight, 0.0), torch.where(valid, d * weight, 0.0)
    return [loss.sum().float(), d.to(s["logprobs"].dtype)]


def _preference(s):
    c = s["case"]
    beta = 0.1
    if own:
        from greyhound_b200.nn.functional import preference_loss

        loss, rewards = preference_loss(s["logprobs"], s["ref"], mask=s["mask"], cu_seqlens=s["cu"], beta=beta, loss_type=c["kind"],
                                        label_smoothing=c["smoothing"] if c["kind"] == "sigmoid" else 0.0,
                                        length_normalized=c["normalized"], return_rewards=True)
        return [loss.detach(), rewards.chosen, rewards.rejected, *torch.autograd.grad(loss, s["logprobs"])]
    seq, valid, n = _token_rows(s)
    # 64 bits: long sums of differences
    diff = torch.where(valid, s["logprobs"].detach().double() - s["ref"].double(), 0.0)
    per = torch.zeros(len(n), dtype=torch.float64, device=diff.device).index_add_(0, seq.reshape(-1), diff.reshape(-1))
    each = 1.0 / n.clamp(min=1).double() if c["normalized"] else torch.ones_like(per)
    per = per * each
    pairs = len(n) // 2
    h = per[:pairs] - per[pairs:]
    if c["kind"] == "sigmoid":
        e = c["smoothing"]
        loss = (1 - e) * (1 + (-beta * h).exp()).log() + e * (1 + (beta * h).exp()).log()
        dh = beta * (e / (1 + (-beta * h).exp()) - (1 - e) / (1 + (beta * h).exp()))
    elif c["kind"] == "hinge":
        loss = (1 - beta * h).clamp(min=0)
        dh = torch.where(beta * h < 1, -beta, 0.0)
    else:
        loss = (h - 1 / (2 * beta)) ** 2
        dh = 2 * (h - 1 / (2 * beta))
    coef = torch.cat([dh, -dh]) * each / pairs
    grad = torch.where(valid, coef[seq], 0.0)
    return [loss.mean().float(), (beta * per[:pairs]).float(), (beta * per[pairs:]).float(), grad.to(s["logprobs"].dtype)]


def _clip(s):
    grads, out = s["grads"], s["out"]
    if own:
        from greyhound_b200.nn.utils import clip_by_global_norm

        _, norm = clip_by_global_norm(grads, s["max_norm"], out=out)
        return [norm, s["flat"]]
    # 64 bits: a sum over every gradient
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    _ = [o.copy_(g.float() * scale) for g, o in zip(grads, out)]
    return [norm.float(), s["flat"]]


RUN = {"linear_logprobs": _linear_logprobs, "policy": _policy, "preference": _preference, "clip": _clip}


def run(state):
    return RUN[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    if case["op"] == "linear_logprobs":
        e = BYTES[case["dtype"]]
        n, d, v = case["rows"], case["hidden"], case["vocab"]
        forward = (n + v) * d * e + 12 * n
        return {"bytes": forward + ((n + v) * d * e + 4 * n if case["train"] else 0), "flops": (6 if case["train"] else 2) * n * d * v}
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        # below the limit the norm is all there is; over it every gradient is read again and written
        return {"bytes": n * BYTES[case["dtype"]] * (1 if case["in_place"] else 3), "flops": n * (2 if case["in_place"] else 3)}
    # half the padded positions hold no token, whose mask alone has to be read; all gradients are written
    e = BYTES[case["dtype"]]
    count = case["seqs"] if case["op"] == "policy" else 2 * case["pairs"]
    tokens = count * case["longest"] * 9 // 16
    slots = tokens if case["packed"] else count * case["longest"]
    if case["op"] == "policy":
        read = 2 * e + (e if case["kl"] else 0) + (4 if case["per_token"] else 0)
        return {"bytes": tokens * read + slots * (e + (0 if case["packed"] else 1)) + 4 * count, "flops": 20 * tokens}
    return {"bytes": tokens * 2 * e + slots * (e + (0 if case["packed"] else 1)) + 8 * count, "flops": 4 * tokens}


# --------------------------------------------------------------------------
# The definitions, in 64 bits


def _exact_linear_logprobs(s):
    c = s["case"]
    w = s["weight"].detach().double()
    weight_grad = torch.zeros_like(w) if c["train"] else None
    logprobs, input_grad = [], []
    block = max(1, (1 << 27) // c["vocab"])
    for a in range(0, c["rows"], block):
        h = s["inputs"].detach()[a : a + block].double()
        t, g = s["index"][a : a + block], s["grad"][a : a + block].double()
        logp = torch.log_softmax(h @ w.T / c["temperature"], dim=1)
        on = t != IGNORE
        at = t.clamp(min=0)[:, None]
        logprobs.append(torch.where(on, logp.gather(1, at)[:, 0], 0.0))
        if c["train"]:
            g = (torch.where(on, g, 0.0) / c["temperature"])[:, None]
            d = torch.zeros_like(logp).scatter_(1, at, g) - g * logp.exp()
            input_grad.append(d @ w)
            weight_grad += d.T @ h
    if not c["train"]:
        return torch.cat(logprobs)
    return [torch.cat(logprobs), torch.cat(input_grad), weight_grad]


def _split(s, t):
    """A batch's sequences, each its valid values, and a function that lays such a list out like the batch."""
    if s["cu"] is None:
        keep = s["mask"]
        n = keep.sum(1).tolist()
        values = list(t.double()[keep].split(n))
        return values, lambda parts: torch.zeros(t.shape, dtype=torch.float64, device=t.device).masked_scatter_(keep, torch.cat(parts))
    return list(t.double().split((s["cu"][1:] - s["cu"][:-1]).tolist())), torch.cat


def _exact_policy(s):
    c = s["case"]
    lp, lay = _split(s, s["logprobs"].detach())
    old, ref = _split(s, s["old"])[0], _split(s, s["ref"])[0]
    adv = _split(s, s["advantages"])[0] if c["per_token"] else [s["advantages"][i].double() for i in range(len(lp))]
    total, filled = sum(x.numel() for x in lp), sum(x.numel() > 0 for x in lp)
    loss, grads = torch.zeros((), dtype=torch.float64, device="cuda"), []
    for x, o, f, a in zip(lp, old, ref, adv):
        x = x.clone().requires_grad_(True)
        ratio = torch.exp(x - o)
        term = -torch.minimum(ratio * a, ratio.clamp(1 - 0.2, 1 + 0.28) * a)
        if c["kl"]:
            term = term + c["kl"] * (torch.exp(f - x) - (f - x) - 1)
        scale = {"sum": 1.0, "mean": 1.0 / max(total, 1), "sequence_mean": 1.0 / (max(x.numel(), 1) * max(filled, 1))}[c["reduction"]]
        part = term.sum() * scale
        grads.append(torch.autograd.grad(part, x)[0] if x.numel() else x.detach())
        loss = loss + part.detach()
    return [loss, lay(grads)]


def _exact_preference(s):
    c = s["case"]
    lp, lay = _split(s, s["logprobs"].detach())
    ref = _split(s, s["ref"])[0]
    lp = [x.clone().requires_grad_(True) for x in lp]
    margins = [(x - f).sum() / (max(x.numel(), 1) if c["normalized"] else 1) for x, f in zip(lp, ref)]
    pairs = len(lp) // 2
    h = torch.stack(margins[:pairs]) - torch.stack(margins[pairs:])
    if c["kind"] == "sigmoid":
        soft = torch.nn.functional.softplus
        loss = ((1 - c["smoothing"]) * soft(-0.1 * h) + c["smoothing"] * soft(0.1 * h)).mean()
    elif c["kind"] == "hinge":
        loss = torch.relu(1 - 0.1 * h).mean()
    else:
        loss = (h - 5.0).square().mean()
    grads = torch.autograd.grad(loss, lp)
    rewards = 0.1 * torch.stack(margins).detach()
    return [loss.detach(), rewards[:pairs], rewards[pairs:], lay(list(grads))]


def _exact_clip(s):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        total += torch.dot(g.double().flatten(), g.double().flatten())
    norm = total.sqrt()
    scale = min(1.0, s["max_norm"] / (norm.item() + 1e-6))
    pieces = [torch.nn.functional.pad(g.double().flatten() * scale, (0, -g.numel() % 8)) for g in s["grads"]]
    return [norm, torch.cat(pieces)]


EXACT = {"linear_logprobs": _exact_linear_logprobs, "policy": _exact_policy, "preference": _exact_preference, "clip": _exact_clip}


def exact(case, seed):
    if case["op"] in ("policy", "preference") and _sequences(case) > 2048:
        return None
    return EXACT[case["op"]](prepare(case, seed))


def _sequences(case):
    return case["seqs"] if case["op"] == "policy" else 2 * case["pairs"]
