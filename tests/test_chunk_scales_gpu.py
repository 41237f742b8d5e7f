"""int8 pages whose scales are far apart: a page's scale counts for the tokens that see the page alone."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu


def check(c, new, ctx, q, qt, kernel):
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new), max_len=max(c["total"]),
                k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)
    at = 0
    for b, n in enumerate(new):
        v = rows_of(c, "v", b)
        want = attention64(q[at:at + n], rows_of(c, "k", b), v, ctx[b])
        # the largest value that a token sees so far, per KV head
        most = v.abs().amax(-1).cummax(0).values[ctx[b]:ctx[b] + n].repeat_interleave(q.shape[1] // v.shape[1], 1)
        err = (o[at:at + n].double() - want).abs().amax(-1) / most.clamp(min=1e-30)
        assert err.max().item() <= tolerance(qt), (b, err.max().item())
        at += n


@pytest.mark.parametrize("kernel", [kvb.Kernel.auto, kvb.Kernel.simt])
@pytest.mark.parametrize("D,page", [(64, 8), (128, 16), (128, 64)])
@pytest.mark.parametrize("new,ctx", [([40], [40]), ([20, 3], [300, 1500]), ([200], [100])])
@pytest.mark.parametrize("big", [1e3, 1e5, 1e8, 1e30, 1e36])
def test_a_later_pages_large_scale_does_not_reach_earlier_tokens(kernel, D, page, new, ctx, big):
    """(fp32 outputs: the larger values would not fit fp16.)"""
    c = make_cache(new, ctx, 2, D, page, I8, 3)
    for b, (n, x) in enumerate(zip(new, ctx)):
        blk = c["table"][b, (x + n - 1) // page].long()  # the last page
        c["vs"][blk, 0] *= big
    check(c, new, ctx, make_q(sum(new), 8, D, F32, 4), F32, kernel)


@pytest.mark.parametrize("kernel", [kvb.Kernel.auto, kvb.Kernel.simt])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("small", [1e-3, 1e-6, 1e-9])
def test_small_scales_before_a_larger_one_fp16(kernel, D, small):
    new, ctx, page = [60, 4], [70, 900], 16
    c = make_cache(new, ctx, 2, D, page, I8, 3)
    # values of ordinary size, but for the last page's, 1 / small times the others: rows before it keep 11 bits
    for b, (n, x) in enumerate(zip(new, ctx)):
        last = c["table"][b, (x + n - 1) // page].long()
        c["vs"][last] *= min(1 / small, 6e4)
        others = c["table"][b, :(x + n - 1) // page].long()
        c["vs"][others] *= min(1.0, 6e4 * small) if small < 1e-4 else 1.0
    q = make_q(sum(new), 8, D, F16, 4)
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=60, max_len=904, k_scale=c["ks"],
                v_scale=c["vs"], kernel=kernel)
    at = 0
    for b, n in enumerate(new):
        v = rows_of(c, "v", b)
        want = attention64(q[at:at + n], rows_of(c, "k", b), v, ctx[b])
        most = v.abs().amax(-1).cummax(0).values[ctx[b]:ctx[b] + n].repeat_interleave(4, 1)
        # an fp16 output below 2^-14 has a step of 2^-24
        err = ((o[at:at + n].double() - want).abs().amax(-1) - 2.0 ** -25).clamp(min=0) / most
        assert err.max().item() <= tolerance(F16), b
        at += n


@pytest.mark.parametrize("kernel", [kvb.Kernel.auto, kvb.Kernel.simt])
@pytest.mark.parametrize("qt", [F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_scales_of_either_sign_and_zero(kernel, qt, D):
    new, ctx = [60, 4, 1], [70, 900, 0]
    c = make_cache(new, ctx, 2, D, 16, I8, 3)
    c["vs"][::3] *= -1
    c["ks"][::2] *= -1
    c["vs"][1::5] = 0
    check(c, new, ctx, make_q(sum(new), 8, D, qt, 4), qt, kernel)
    c["vs"][:] = -c["vs"].abs()
    check(c, new, ctx, make_q(sum(new), 8, D, qt, 5), qt, kernel)
