"""Inputs and 64-bit results for the serving-step operators' GPU tests (plain loops over sequences)."""
import math

import numpy as np
import torch

F32, F16, I8 = torch.float32, torch.float16, torch.int8


def make_cache(new, ctx, Hkv, D, page, kv, seed, slack=2):
    """Pools whose dead slots and unused pages hold NaN (int8: any bits, NaN scales on unused pages)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = [n + c for n, c in zip(new, ctx)]
    pages = [-(-t // page) for t in total]
    num_blocks = sum(pages) + slack
    perm = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
    width = max(pages + [1])
    table = torch.full((len(new), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    live = torch.zeros(num_blocks, page, dtype=torch.bool, device="cuda")
    for b, t in enumerate(total):
        for j in range(pages[b]):
            live[table[b, j].long(), :min(page, t - j * page)] = True
    c = dict(table=table, num_blocks=num_blocks, total=total, page=page, live=live)
    shape = (num_blocks, Hkv, page, D)
    for x in "kv":
        if kv is I8:
            c[x] = torch.randint(-127, 128, shape, dtype=I8, device="cuda", generator=g)
            c[x + "s"] = torch.empty(num_blocks, Hkv, device="cuda").uniform_(1e-4, 1 / 127, generator=g)
            c[x + "s"][~live.any(1)] = float("nan")
        else:
            y = torch.empty(shape, device="cuda").uniform_(-1, 1, generator=g).to(kv)
            c[x] = torch.where(live[:, None, :, None], y, float("nan")).contiguous()
            c[x + "s"] = None
    return c


def rows_of(c, x, b):
    """Sequence b's keys or values [total][Hkv][D] in float64."""
    t = c["total"][b]
    ids = c["table"][b, :-(-t // c["page"])].long()
    y = c[x][ids].double()
    if c[x + "s"] is not None:
        y = y * c[x + "s"][ids].double()[:, :, None, None]
    return y.permute(0, 2, 1, 3).reshape(-1, y.shape[1], y.shape[3])[:t]


def attention64(q, k, v, first):
    """q [n][H][D], k and v [L][Hkv][D] in float64; query i at position first + i."""
    n, H, D = q.shape
    G = H // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / math.sqrt(D)
    seen = torch.arange(k.shape[0], device="cuda")[None] <= first + torch.arange(n, device="cuda")[:, None]
    s = torch.where(seen[None], s, -math.inf)
    p = torch.softmax(s, -1)
    terms = torch.where(seen[None, :, :, None], v.permute(1, 0, 2)[:, None], 0.0) if not torch.isfinite(v).all() else None
    if terms is not None:  # a value that is not seen takes no part, whatever it is
        return torch.einsum("hij,hijd->ihd", p, terms)
    return torch.einsum("hij,jhd->ihd", p, v)


def starts(new):
    return torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device="cuda")


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def make_q(T, H, D, dtype, seed, pad=0):
    """Query rows with `pad` more elements between tokens (NaN, never read)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.full((T, H * D + pad), float("nan"), dtype=dtype, device="cuda")
    q[:, :H * D] = torch.empty(T, H * D, device="cuda").uniform_(-1, 1, generator=g).to(dtype)
    return q[:, :H * D].view(T, H, D)


def tolerance(q_dtype):
    """|out - exact| for values of at most 1. fp32: the reference's kernel tolerance on inputs of this
    distribution. fp16: the output's rounding and the probabilities' are each off by at most half a
    step, 2^-11 relative, of terms that sum to at most 1; the rest is fp32."""
    return 2e-5 if q_dtype is F32 else 2 * 2.0 ** -11 + 2e-5
