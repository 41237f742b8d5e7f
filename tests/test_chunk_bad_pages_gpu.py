"""Block ids outside the pool in attention of several new tokens: the tokens that see the page become NaN,
whichever query tile, unit or piece they are in, and no other row changes."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu
AUTO, SIMT = kvb.Kernel.auto, kvb.Kernel.simt


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F16, I8), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 4, 64, 16), (8, 2, 128, 64), (4, 1, 128, 256)])
@pytest.mark.parametrize("new,ctx,at", [([300], [100], 250), ([300], [100], 399), ([200, 3], [0, 900], 130),
                                        ([64], [3000], 3040), ([70], [3000], 1500)])
@pytest.mark.parametrize("bad_id", [-1, None])
def test_a_bad_page_reaches_the_tokens_that_see_it(kernel, qt, kv, H, Hkv, D, page, new, ctx, at, bad_id):
    c = make_cache(new, ctx, Hkv, D, page, kv, seed=3)
    q = make_q(sum(new), H, D, qt, 4)
    want = torch.cat([attention64(q[x:x + n], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
                      for b, (x, n) in enumerate(zip(starts(new).tolist(), new))])
    c["table"][0, at // page] = c["num_blocks"] if bad_id is None else bad_id
    a = ops.PagedPrefill()

    def run():
        return a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new),
                       max_len=max(c["total"]), k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)

    o = run()
    assert a.error_flag() == 2
    first = max(0, at // page * page - ctx[0])  # the first token of sequence 0 that sees the page
    assert o[first:new[0]].isnan().all()
    fine = torch.ones(sum(new), dtype=torch.bool, device="cuda")
    fine[first:new[0]] = False
    assert (o[fine].double() - want[fine]).abs().max().item() <= tolerance(qt) if fine.any() else True
    for _ in range(5):
        assert torch.equal(run()[fine], o[fine])


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F16, I8), (F32, I8)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,ctx,at", [([200], [300], 400), ([60], [3000], 3030), ([256], [0], 130)])
def test_what_ran_before_does_not_show_in_the_rows_beside_nan_ones(qt, kv, D, new, ctx, at):
    """Shared memory that the refused page was not loaded into holds keys of the call before, of any size."""
    c = make_cache(new, ctx, 2, D, 16, kv, seed=3)
    q = make_q(sum(new), 4, D, qt, 4) * 3
    c["table"][0, at // 16] = -1
    x = make_cache([500] * 4, [200] * 4, 2, D, 16, kv, seed=6)
    other = make_q(2000, 4, D, qt, 5)
    if kv is not I8:
        keys = [x["k"].nan_to_num(0.0) * s for s in (0.001, 3.0, 3000.0)]
    else:
        keys = [x["k"] // 2, x["k"], x["k"] * 0]
    a = ops.PagedPrefill()
    outs = []
    for i in range(12):
        a.chunk(other, keys[i % 3], x["v"], x["table"], ints(x["total"]), starts([500] * 4), max_new=500, max_len=700,
                k_scale=x["ks"], v_scale=x["vs"])
        outs.append(a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new),
                            max_len=c["total"][0], k_scale=c["ks"], v_scale=c["vs"]))
    first = at // 16 * 16 - ctx[0]
    assert outs[0][:first].isfinite().all() and outs[0][first:].isnan().all()
    for o in outs[1:]:
        assert torch.equal(o[:first], outs[0][:first])
