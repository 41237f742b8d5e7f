"""Attention of several new tokens per sequence where the scores are far apart: a row's running
reference moves after its first key tile, inside a tile, past folded sums and between the pieces of a
cut unit. Against 64 bits.

All products of q and k are multiples of 2^-12 whose absolute sums stay below 2^12 (fp16 queries:
2^-6 and 2^18), so every score is exact in fp32 in whatever order it is added up, and the tolerance is
that of scores near 0.
"""
import math

import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu
AUTO, SIMT = kvb.Kernel.auto, kvb.Kernel.simt


def grid(shape, lo, hi, step, g):
    return torch.randint(lo, hi + 1, shape, device="cuda", generator=g).float() * step


def make_queries(T, H, D, qt, seed):
    """First component 4, the others multiples of 1/8 up to 1; fp32 ones have bits that no fp16 holds."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = grid((T, H, D), -8, 8, 0.125, g)
    q[:, :, 0] = 4.0
    if qt is F32:
        q += grid((T, H, D), -15, 15, 2.0 ** -9, g)
    return q.to(qt)


def set_keys(c, b, levels, D, kv, seed):
    """Sequence b's keys: components that score about 0, and a first one that puts position j levels[j]
    log2 units above that (against 4.0 in q)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    L, page, Hkv = len(levels), c["page"], c["k"].shape[1]
    first = torch.tensor(levels, dtype=torch.float64, device="cuda") * math.sqrt(D) / (4 * math.log2(math.e))
    ids = c["table"][b, :-(-L // page)].long()
    pos = torch.arange(L, device="cuda")
    at = (ids[pos // page], slice(None), pos % page)
    if kv is I8:  # scales of 8 and 4
        scale = torch.where(torch.arange(len(ids), device="cuda") % 3 == 0, 4.0, 8.0)
        if max(map(abs, levels)) * math.sqrt(D) / (4 * math.log2(math.e)) > 4 * 127:
            scale[:] = 8.0
        c["ks"][ids] = scale[:, None]
        k = grid((L, Hkv, D), -1, 1, 1.0, g)
        k[:, :, 0] = (first / scale[pos // page]).round().clamp(-127, 127).float()[:, None]
    else:
        k = grid((L, Hkv, D), -8, 8, 0.125, g)
        k[:, :, 0] = (first * 8).round().float()[:, None] / 8
    c["k"][at] = k.to(kv)


def check(new, ctx, levels, H, Hkv, D, page, qt, kv, *, seed=1, kernel=AUTO):
    """levels(position, tokens of the sequence): log2 units."""
    c = make_cache(new, ctx, Hkv, D, page, kv, seed)
    for b, total in enumerate(c["total"]):
        set_keys(c, b, [levels(j, total) for j in range(total)], D, kv, seed + b)
    q = make_queries(sum(new), H, D, qt, seed)
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new), max_len=max(c["total"]),
                k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)
    assert a.error_flag() == 0
    at = 0
    for b, n in enumerate(new):
        if n:
            want = attention64(q[at:at + n], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
            err = (o[at:at + n].double() - want).abs().max().item()
            assert err <= tolerance(qt), (b, n, ctx[b], err)
        at += n


@pytest.mark.parametrize("kv", [F16, I8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [10, 20, 50, 150, 400])
def test_fp32_queries_reference_rises_inside_key_tiles(kv, D, step):
    """Split probabilities that were written already follow the reference: every 32 keys it rises."""
    check([70, 3], [500, 4000], lambda j, n: min(step * (j // 32), 450), 8, 2, D, 16, F32, kv)
    check([70, 3], [500, 4000], lambda j, n: min(step * (j // 32 % 4), 450), 8, 2, D, 128, F32, kv)


ONE_IN_32 = list(range(32))


@pytest.mark.parametrize("kind", ["pages", "int8 pages", "prompt"])
@pytest.mark.parametrize("up", [126, 128.2, 130, 200, 300, 400, 500])
def test_one_key_far_above_the_first_tile_counts_wherever_it_lies(kind, up):
    """Head dim 64: part of the exponentials are a polynomial, by the key's place among 32. A batch of 32
    sequences, the key of sequence b at position 128 + b, `up` log2 units above the others."""
    H, Hkv, D, n = 4, 2, 64, 12
    new, ctx = [n] * 32, [200] * 32
    kv = I8 if kind == "int8 pages" else F16
    if kind != "prompt":
        c = make_cache(new, ctx, Hkv, D, 64, kv, 5)
        for b in ONE_IN_32:
            set_keys(c, b, [up if j == 128 + b else 0.0 for j in range(212)], D, kv, b)
        q = make_queries(n * 32, H, D, F16, 6)
        a = ops.PagedPrefill()
        o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=n, max_len=212,
                    k_scale=c["ks"], v_scale=c["vs"])
        for b in ONE_IN_32:
            want = attention64(q[n * b:n * (b + 1)], rows_of(c, "k", b), rows_of(c, "v", b), 200)
            assert (o[n * b:n * (b + 1)].double() - want).abs().max().item() <= tolerance(F16), b
        return
    c = make_cache([212] * 32, [0] * 32, Hkv, D, 64, F16, 5)  # the same rows, packed
    for b in ONE_IN_32:
        set_keys(c, b, [up if j == 128 + b else 0.0 for j in range(212)], D, F16, b)
    k, v = (torch.cat([rows_of(c, x, b) for b in ONE_IN_32]) for x in "kv")
    q = make_queries(212 * 32, H, D, F16, 6)
    o = ops.PagedPrefill().prompt(q, k.half(), v.half(), starts([212] * 32), max_len=212)
    for b in ONE_IN_32:
        x = slice(212 * b, 212 * (b + 1))
        assert (o[x].double() - attention64(q[x], k[x], v[x], 0)).abs().max().item() <= tolerance(F16), b


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", [F16, I8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_infinite_or_nan_score_makes_the_row_nan(D, kv, bad):
    """... in a later key tile, at every place among 32."""
    new, ctx = [3] * 32, [300] * 32
    c = make_cache(new, ctx, 1, D, 16, kv, 7)
    for b in ONE_IN_32:
        p = 128 + b
        if kv is I8:
            c["k"][c["table"][b, p // 16].long(), 0, :, :] = 1
            c["ks"][c["table"][b, p // 16].long(), 0] = bad
        else:
            c["k"][c["table"][b, p // 16].long(), 0, p % 16, 0] = bad
    q = make_queries(96, 2, D, F16, 6).abs()
    o = ops.PagedPrefill().chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=3, max_len=303,
                                 k_scale=c["ks"], v_scale=c["vs"])
    assert o.isnan().all()


def lowest(c, b, positions, kv):
    """Keys whose score is -inf for queries without a negative or zero component."""
    page = c["page"]
    for p in positions:
        blk = c["table"][b, p // page].long()
        if kv is I8:  # whole pages
            c["k"][blk], c["ks"][blk] = -1, float("inf")
        else:
            c["k"][blk, :, p % page, :] = -1.0
            c["k"][blk, :, p % page, 0] = -float("inf")


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F16, I8), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("level", [0, -12, -20, -30, -80, -200])
@pytest.mark.parametrize("new,ctx,dead", [([5], [400], range(128)), ([130], [256], range(160)), ([3], [400], range(48)),
                                          ([3], [6000], range(2048)), ([3], [6000], range(1024, 4096))])
def test_a_first_key_tile_of_infinitely_low_scores(qt, kv, D, level, new, ctx, dead):
    """The row's reference is set by the first score that is finite, however low it lies."""
    c = make_cache(new, ctx, 2, D, 16, kv, 3)
    set_keys(c, 0, [float(level)] * c["total"][0], D, kv, 4)
    lowest(c, 0, dead, kv)
    q = make_queries(sum(new), 8, D, qt, 5).abs().clamp(min=0.125)
    a = ops.PagedPrefill()
    for kernel in (AUTO, SIMT):
        o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new), max_len=c["total"][0],
                    k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)
        want = attention64(q, rows_of(c, "k", 0), rows_of(c, "v", 0), ctx[0])
        assert (o.double() - want).abs().max().item() <= tolerance(qt)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_prompt_whose_first_keys_score_infinitely_low(dt, D):
    """Tokens that see no other key have no softmax (NaN); the others are the mean over the rest."""
    c = make_cache([500], [0], 2, D, 16, F32, 3)
    set_keys(c, 0, [-40.0] * 500, D, F32, 4)
    lowest(c, 0, range(140), F32)
    k, v = (rows_of(c, x, 0).to(dt) for x in "kv")
    q = make_queries(500, 8, D, dt, 5).abs().clamp(min=0.125)
    for kernel in (AUTO, SIMT):
        o = ops.PagedPrefill().prompt(q, k, v, starts([500]), max_len=500, kernel=kernel)
        want = attention64(q, k.double(), v.double(), 0)
        assert o[:140].isnan().all() and want[:140].isnan().all()
        assert (o[140:].double() - want[140:]).abs().max().item() <= tolerance(dt)


TYPES = [(F16, F16), (F32, F16), (F16, I8), (F32, I8), (F32, F32), (F16, F32)]


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [10, 50, 150, 400])
@pytest.mark.parametrize("every", [1, 40, 128, 200])
def test_rising_scores(kernel, qt, kv, D, step, every):
    """... from key to key, tile to tile and in between, in whole and cut units."""
    check([140, 2], [600, 5000], lambda j, n: min(step * (j // every), 450), 8, 2, D, 64, qt, kv, kernel=kernel)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [-10, -150, -400])
def test_falling_scores(kernel, qt, kv, D, step):
    check([140, 2], [600, 5000], lambda j, n: max(step * (j // 100), -450), 8, 2, D, 64, qt, kv, kernel=kernel)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("up", [15, 60, 400])
def test_single_high_scores(kernel, qt, kv, D, up):
    """One key of every 301, at changing places of the tiles: the later ones a little higher."""
    check([140, 2], [600, 5000], lambda j, n: up + j / 200 if j % 301 == 300 else 0.0, 8, 2, D, 64, qt, kv, kernel=kernel)


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F16, I8), (F32, I8)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("every,step", [(1000, 10), (2500, 60), (128, 3)])
def test_rising_scores_over_folded_sums(qt, kv, D, every, step):
    """CTAs that take more than 64 key tiles of a unit (38 k keys by 64 heads over at most 148 CTAs are 130 tiles each):
    the sums that left tensor memory follow the reference."""
    check([250, 256], [19000, 18800], lambda j, n: min(step * (j // every), 450), 64, 64, D, 128, qt, kv)
