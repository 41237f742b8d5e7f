"""Attention of several new tokens per sequence (kvb_paged_chunk_async, kvb_prompt_async) on the GPU
against 64-bit attention. Dead slots and unused pages hold NaN throughout."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu
AUTO, SIMT = kvb.Kernel.auto, kvb.Kernel.simt


def run_chunk(new, ctx, H, Hkv, D, page, qt, kv, *, seed=1, kernel=AUTO, pad=0, max_new=None, max_len=None):
    c = make_cache(new, ctx, Hkv, D, page, kv, seed)
    q = make_q(sum(new), H, D, qt, seed + 1, pad)
    a = ops.PagedPrefill()
    out = torch.full((sum(new) + 3, H, D), 7.0, dtype=qt, device="cuda")  # three rows behind the last sequence
    qq = torch.cat([q, q.new_full((3, H, D), float("nan"))]) if not pad else q
    o = a.chunk(qq, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max_new or max(new),
                max_len=max_len or max(c["total"]), k_scale=c["ks"], v_scale=c["vs"],
                out=out if not pad else None, kernel=kernel)
    if not pad:
        assert (out[sum(new):] == 7.0).all()
    assert a.error_flag() == 0
    at = 0
    for b, n in enumerate(new):
        if n:
            want = attention64(q[at:at + n], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
            err = (o[at:at + n].double() - want).abs().max().item()
            assert err <= tolerance(qt), (b, n, ctx[b], err)
        at += n


TYPES = [(F16, F16), (F32, F16), (F16, I8), (F32, I8), (F32, F32), (F16, F32)]
HEADS = [(32, 8, 128), (8, 8, 64), (12, 2, 128), (7, 1, 64), (64, 1, 128)]


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("H,Hkv,D", HEADS)
def test_chunk_ragged(kernel, qt, kv, H, Hkv, D):
    run_chunk([1, 5, 0, 33, 130, 1], [0, 123, 77, 0, 61, 300], H, Hkv, D, 16, qt, kv, kernel=kernel)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("page", [1, 8, 24, 32, 64, 128, 256])
def test_chunk_pages(qt, kv, page):
    run_chunk([9, 70], [250, 127], 8, 2, 128, page, qt, kv, seed=page)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1], [1]), ([1], [127]), ([1], [128]), ([2], [126]), ([3], [5000]),
                                     ([64], [1000]), ([65], [63]), ([200], [1025]), ([1, 2], [8191, 3])])
def test_chunk_lengths_and_split_keys(qt, kv, new, ctx):
    run_chunk(new, ctx, 8, 2, 128, 64, qt, kv, seed=len(new) + ctx[0])


@pytest.mark.parametrize("qt,kv", TYPES)
def test_chunk_bounds_larger_than_the_lengths(qt, kv):
    run_chunk([3, 40], [500, 2], 8, 2, 128, 32, qt, kv, max_new=500, max_len=20000)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_chunk_many_units(qt, kv):
    # more units than CTAs, so that CTAs take several
    n = 330 if kv is not F32 and qt is F16 else 150
    run_chunk([n + i for i in range(6)], [90 * i for i in range(6)], 32, 16, 64, 16, qt, kv)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B", [500, 1300])
def test_chunk_many_sequences(qt, kv, B):
    # more sequences than a CTA has threads, some without new tokens
    new = [i % 4 for i in range(B)]
    ctx = [(7 * i) % 90 + (2000 if i % 97 == 0 else 0) for i in range(B)]
    run_chunk(new, ctx, 4, 2, 64, 16, qt, kv)


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F16, I8), (F32, I8)])
def test_chunk_long_keys_few_ctas(qt, kv):
    # so many units that each CTA takes long runs of key tiles: the running sums leave tensor memory
    run_chunk([256, 250], [20000, 9000], 32, 32, 64, 128, qt, kv)


@pytest.mark.parametrize("qt", [F16, F32])
def test_chunk_query_stride(qt):
    run_chunk([20, 7], [40, 0], 8, 2, 128, 16, qt, F16, pad=64)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx", [0, 120, 3000])
def test_nonfinite_values_reach_only_the_tokens_that_see_them(kernel, qt, kv, D, ctx):
    new, H, Hkv, page = [40], 4, 2, 16
    c = make_cache(new, [ctx], Hkv, D, page, kv, seed=5)
    q = make_q(40, H, D, qt, 6)

    def poke(x, p, d, val):
        blk, r = int(c["table"][0, p // page]), p % page
        if kv is I8:
            c[x + "s"][blk, 0] = val  # the whole page of head 0
        else:
            c[x][blk, 0, r, d] = val

    poke("v", ctx + 33, 5, float("inf"))
    poke("v", ctx + 37, 6, float("nan"))
    poke("k", ctx + 38, 7, float("nan"))
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=40, max_len=ctx + 40,
                k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)
    want = attention64(q, rows_of(c, "k", 0), rows_of(c, "v", 0), ctx)
    first = ctx + 33 if kv is not I8 else (ctx + 33) // page * page  # the first token that sees one
    assert torch.isfinite(o[:max(0, first - ctx)]).all()
    # head 0's group sees them, the others do not
    assert torch.isfinite(o[:, H // 2:]).all()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(o)) and torch.equal(want.isnan(), o.isnan())
    assert (torch.where(fine, o.double() - want, 0.0).abs().max().item()) <= tolerance(qt)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("max_len", [400, 30000])
def test_refused_sequences_become_nan_and_leave_the_others(qt, kv, max_len):
    new, ctx, H, Hkv, D, page = [5, 4, 3, 6, 2, 7], [60, 0, 30, 10, 40, 100], 8, 2, 128, 16
    c = make_cache(new, ctx, Hkv, D, page, kv, seed=9)
    q = make_q(sum(new), H, D, qt, 10)
    total = ints(c["total"])
    total[1] = -1                      # refused by the plan
    total[2] = 2                       # fewer than its new tokens
    total[4] = 16 * c["table"].shape[1] + 1   # beyond the table
    c["table"][3, 0] = c["num_blocks"]  # outside the pool
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], total, starts(new), max_new=7, max_len=max_len, k_scale=c["ks"],
                v_scale=c["vs"])
    assert a.error_flag() == 3 and a.error_flag() == 0
    cu = starts(new).tolist()
    for b in range(6):
        got = o[cu[b]:cu[b + 1]]
        if b in (0, 5):
            want = attention64(q[cu[b]:cu[b + 1]], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
            assert (got.double() - want).abs().max().item() <= tolerance(qt)
        else:
            assert got.isnan().all(), b
    # more new tokens than max_new, a total above max_len, rows outside the packed step
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=6, max_len=64, k_scale=c["ks"],
                v_scale=c["vs"])
    assert a.error_flag() & 1
    assert o[cu[5]:].isnan().all() and o[:cu[1]].isnan().all()
    cu_bad = starts(new)
    cu_bad[6] = 1000
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), cu_bad, max_new=2000, max_len=max_len,
                k_scale=c["ks"], v_scale=c["vs"])
    assert a.error_flag() & 1 and o[cu[5]:].isnan().all() and o[:cu[1]].isfinite().all()


@pytest.mark.parametrize("kv", [F32, F16, I8])
def test_one_new_token_is_the_decode_step(kv):
    new, ctx = [1, 1, 1], [700, 0, 64]
    c = make_cache(new, ctx, 2, 128, 16, kv, seed=4)
    q = make_q(3, 8, 128, F32, 5)
    d, a, lens = ops.PagedDecoder(), ops.PagedPrefill(), ints(c["total"])
    x = d(q, c["k"], c["v"], c["table"], lens, 701, k_scale=c["ks"], v_scale=c["vs"])
    y = a.chunk(q, c["k"], c["v"], c["table"], lens, starts(new), max_new=1, max_len=701, k_scale=c["ks"], v_scale=c["vs"])
    assert (x - y).abs().max().item() <= 2 * tolerance(F32)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("new", [[1], [130, 1, 0, 257, 64], [128], [1000, 3]])
def test_prompt(kernel, dt, H, Hkv, D, new):
    T = sum(new)
    qkv = make_q(T + 2, H + 2 * Hkv, D, dt, 3, pad=8)
    qkv[T:] = float("nan")  # rows behind the last prompt
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    a = ops.PagedPrefill()
    out = torch.full((T + 2, H, D), 7.0, dtype=dt, device="cuda")
    a.prompt(q, k, v, starts(new), max_len=max(new), out=out, kernel=kernel)
    assert a.error_flag() == 0 and (out[T:] == 7.0).all()
    at = 0
    for n in new:
        if n:
            want = attention64(q[at:at + n], k[at:at + n].double(), v[at:at + n].double(), 0)
            assert (out[at:at + n].double() - want).abs().max().item() <= tolerance(dt), n
        at += n


@pytest.mark.parametrize("dt", [F16, F32])
def test_prompts_do_not_see_each_other(dt):
    new = [70, 200, 9]
    q, k, v = (make_q(279, h, 64, dt, 3 + h) for h in (4, 2, 2))
    k[70:270] = float("nan")
    v[70:270] = float("inf")
    a = ops.PagedPrefill()
    o = a.prompt(q, k, v, starts(new), max_len=200)
    assert o[:70].isfinite().all() and o[270:].isfinite().all() and not o[70:270].isfinite().any()


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, I8), (F32, F32)])
def test_a_request_served_step_by_step(qt, kv):
    """plan, append and attention over three steps (a prompt, a chunk, single tokens) of two requests, as
    a server runs them, against attention over everything so far."""
    H, Hkv, D, page, num_blocks, width = 8, 2, 128, 16, 40, 20
    g = torch.Generator(device="cuda").manual_seed(2)
    pool_dtype = kv
    pools = [torch.zeros(num_blocks, Hkv, page, D, dtype=pool_dtype, device="cuda") for _ in range(2)]
    scales = [torch.zeros(num_blocks, Hkv, device="cuda") for _ in range(2)]
    ring = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
    ring_pos = ints([0, num_blocks], torch.int64)
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    lens, err, a = ints([0, 0]), ints([0]), ops.PagedPrefill()
    seen = [[[], []], [[], []]]
    for new in ([100, 37], [30, 1], [1, 1], [1, 0]):
        T = sum(new)
        q = make_q(T, H, D, qt, T)
        k, v = make_q(T, Hkv, D, qt, T + 1), make_q(T, Hkv, D, qt, T + 2)
        p = ops.plan_step(lens, ints(new), table, ring, ring_pos, page_size=page, num_blocks=num_blocks, num_tokens=T,
                          error_word=err)
        if kv is I8:
            ops.append_kv_i8(k, v, *pools, *scales, block_table=table, total_lens=p.total_lens, cu_new=p.cu_new,
                             error_word=err)
        else:
            ops.append_kv(k, v, *pools, slot_map=p.slot_map, error_word=err)
        o = a.chunk(q, *pools, table, p.total_lens, p.cu_new, max_new=max(new), max_len=width * page,
                    k_scale=scales[0] if kv is I8 else None, v_scale=scales[1] if kv is I8 else None)
        assert err.item() == 0 and a.error_flag() == 0
        at = 0
        for b, n in enumerate(new):
            for x, rows in enumerate((k, v)):
                seen[b][x].append(rows[at:at + n].double())
            if n:
                kk, vv = (torch.cat(y) for y in seen[b])
                want = attention64(q[at:at + n], kk, vv, kk.shape[0] - n)
                # int8: a value is off by half a step of its page's scale, at most 1 / 254, once when it
                # is written and once whenever the scale grows (three appends at most to a page here), a score by
                # sqrt(D) times that times the largest |q| and log-weights by the sum: well within
                tol = tolerance(qt) if kv is not I8 else 0.05
                assert (o[at:at + n].double() - want).abs().max().item() <= tol
            at += n
        lens, ring_pos = p.total_lens, p.ring_pos


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F16, I8), (F32, F16), (F32, I8)])
@pytest.mark.parametrize("H,Hkv", [(20, 4), (7, 1), (33, 11)])
def test_results_do_not_depend_on_what_ran_before(qt, kv, H, Hkv):
    """Group sizes that leave rows of the query tile without a token; calls with other values in between."""
    new, ctx = [3, 97, 1, 40], [700, 30, 0, 2500]
    c = make_cache(new, ctx, Hkv, 128, 32, kv, 3)
    q, other = make_q(sum(new), H, 128, qt, 4) * 8, make_q(500, H, 128, qt, 5) * 60
    x = make_cache([500], [40], Hkv, 128, 32, kv, 6)
    a = ops.PagedPrefill()

    def run():
        return a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=97, max_len=2540,
                       k_scale=c["ks"], v_scale=c["vs"])

    first = run()
    for _ in range(10):
        a.chunk(other, x["k"], x["v"], x["table"], ints(x["total"]), starts([500]), max_new=500, max_len=540,
                k_scale=x["ks"], v_scale=x["vs"])
        assert torch.equal(run(), first)


@pytest.mark.parametrize("qt", [F16, F32])
@pytest.mark.parametrize("H,Hkv,D", [(33, 11, 64), (20, 4, 64), (33, 11, 128)])
@pytest.mark.parametrize("new,ctx", [([181, 1], [9591, 133]), ([250, 1, 1, 1], [9244, 100, 133, 250]),
                                     ([84] + [1] * 40, [1000] + [140] * 40)])
def test_scales_stay_until_the_slower_query_tile_has_used_them(qt, H, Hkv, D, new, ctx):
    # Units of one token have rows in one of the two query tiles only; the other one may still be in the unit before.
    for seed in range(6):
        c = make_cache(new, ctx, Hkv, D, 128, I8, seed)
        q = make_q(sum(new), H, D, qt, seed + 1)
        a = ops.PagedPrefill()

        def run():
            return a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new),
                           max_len=max(c["total"]), k_scale=c["ks"], v_scale=c["vs"], kernel=kvb.Kernel.umma)

        first = run()
        for _ in range(30):
            assert torch.equal(run(), first)
        at = 0
        for b, n in enumerate(new):
            want = attention64(q[at:at + n], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
            assert (first[at:at + n].double() - want).abs().max().item() <= tolerance(qt), (seed, b)
            at += n


@pytest.mark.parametrize("kv", [F16, I8])
def test_pools_past_32_bits(kv):
    """Pages whose first value lies more than 2^31 elements into the pool (and 2^32 bytes)."""
    Hkv, D, page, num_blocks = 8, 128, 128, 18000
    pools = [torch.zeros(num_blocks, Hkv, page, D, dtype=kv, device="cuda") for _ in range(2)]
    scales = [torch.zeros(num_blocks, Hkv, device="cuda") for _ in range(2)]
    assert pools[0].numel() > 1 << 31
    new, ids = [200, 129], [[num_blocks - 1, num_blocks - 7], [num_blocks - 3, 5]]
    table = ints(ids)
    T = sum(new)
    q, k, v = make_q(T, 16, D, F16, 1), make_q(T, Hkv, D, F16, 2), make_q(T, Hkv, D, F16, 3)
    total, cu = ints(new), starts(new)
    if kv is I8:
        ops.append_kv_i8(k, v, *pools, *scales, block_table=table, total_lens=total, cu_new=cu)
    else:
        slots = [ids[b][p // page] * page + p % page for b, n in enumerate(new) for p in range(n)]
        ops.append_kv(k, v, *pools, slot_map=ints(slots, torch.int64))
    a = ops.PagedPrefill()
    for kernel in (AUTO, SIMT):
        o = a.chunk(q, *pools, table, total, cu, max_new=200, max_len=200, k_scale=scales[0] if kv is I8 else None,
                    v_scale=scales[1] if kv is I8 else None, kernel=kernel)
        assert a.error_flag() == 0
        for b, (x, n) in enumerate(zip(cu.tolist(), new)):
            c = dict(total=new, page=page, table=table, k=pools[0], v=pools[1], ks=scales[0] if kv is I8 else None,
                     vs=scales[1] if kv is I8 else None)
            want = attention64(q[x:x + n], rows_of(c, "k", b), rows_of(c, "v", b), 0)
            assert (o[x:x + n].double() - want).abs().max().item() <= tolerance(F16)


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F16, I8), (F32, F16)])
def test_captured_steps_on_another_stream(qt, kv):
    """Two captured calls that share the object, replayed at once on two streams, and an eager call."""
    cases = []
    a = ops.PagedPrefill()
    for seed, (new, ctx) in enumerate((([3, 40], [4000, 90]), ([300], [700]))):
        c = make_cache(new, ctx, 2, 128, 16, kv, seed)
        q = make_q(sum(new), 8, 128, qt, seed)
        args = (q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new))
        kw = dict(max_new=max(new), max_len=max(c["total"]), k_scale=c["ks"], v_scale=c["vs"])
        eager = a.chunk(*args, **kw)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        out = torch.zeros_like(eager)
        with torch.cuda.graph(g, stream=stream):
            a.chunk(*args, out=out, **kw)
        cases.append((g, stream, eager, out, args, kw))
    for _ in range(5):
        for g, stream, eager, out, args, kw in cases:
            with torch.cuda.stream(stream):
                out.fill_(0)
                g.replay()
        a.chunk(*cases[0][4], **cases[0][5])
        torch.cuda.synchronize()
        for g, stream, eager, out, args, kw in cases:
            assert torch.equal(out, eager)  # bit for bit, whatever ran beside it


def test_tensors_are_checked():
    c = make_cache([4], [0], 2, 64, 16, F16, seed=1)
    q = make_q(4, 4, 64, F16, 1)
    a = ops.PagedPrefill()
    good = dict(max_new=4, max_len=4)
    args = [q, c["k"], c["v"], c["table"], ints(c["total"]), starts([4])]
    for i, bad in ((0, q.cpu()), (0, q.transpose(0, 1)), (0, q.bfloat16()), (1, c["k"].transpose(1, 2)), (2, c["v"].float()),
                   (3, c["table"].long()), (3, c["table"][0]), (4, ints([4]).long()), (5, starts([4])[:1]), (5, starts([4]).cpu())):
        with pytest.raises(ValueError):
            a.chunk(*[bad if j == i else x for j, x in enumerate(args)], **good)
    with pytest.raises(ValueError):
        a.chunk(*args, **good, out=torch.empty(4, 4, 64, device="cuda"))
    with pytest.raises(ValueError):
        a.chunk(*args, **good, k_scale=torch.ones(2, 3, device="cuda"))
    with pytest.raises(ValueError):
        a.prompt(q, q[:, :2].float(), q[:, :2].float(), starts([4]), max_len=4)
