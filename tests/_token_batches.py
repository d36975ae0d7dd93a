"""Batches of tokens in sequences, padded and packed, for the token losses' tests."""

import torch

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def batch(lengths, dtype, seed, padded, other=None, pad=0, front=0, back=0, left_out=0.2):
    """Random tokens of sequences of such lengths; positions outside them hold NaN, inf and -inf."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = torch.tensor(lengths, device="cuda")
    S = len(lengths)
    if padded:
        L = max(lengths, default=0) + pad
        shape = (S, L)
        inside = torch.arange(L, device="cuda") < n[:, None]
        seq = torch.arange(S, device="cuda")[:, None].expand(S, L)
        cu = None
    else:
        T = sum(lengths) + front + back
        shape = (T,)
        cu = torch.zeros(S + 1, dtype=torch.int64, device="cuda")
        cu[1:] = n.cumsum(0)
        cu += front
        seq = torch.full((T,), -1, device="cuda")
        seq[front : front + sum(lengths)] = torch.repeat_interleave(torch.arange(S, device="cuda"), n)
        inside = seq >= 0
    rnd = lambda: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    valid = inside & (torch.rand(shape, device="cuda", generator=g) >= left_out)
    lp = (-rnd().abs() * 2).to(dtype)
    old = (lp.float() + 0.3 * rnd()).to(other or dtype)
    ref = (lp.float() + 0.5 * rnd()).to(other or dtype)
    adv = rnd()
    junk = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min], device="cuda")
    for t in (lp, old, ref, adv):
        fill = junk[torch.randint(0, 4, shape, device="cuda", generator=g)].to(t.dtype)
        t.copy_(torch.where(valid, t, fill))
    return {"lp": lp, "old": old, "ref": ref, "adv": adv, "mask": valid, "cu": cu, "seq": seq, "S": S,
            "adv_s": torch.randn(S, device="cuda", generator=g)}
