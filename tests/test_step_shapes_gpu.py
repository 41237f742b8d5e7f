"""Calls of the serving-step operators at the smallest shapes, and rows of one head in any layout."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("B", [0, 3])
def test_a_step_without_tokens(qt, kv, B):
    c = make_cache([0] * B + [5], [20] * B + [0], 2, 64, 16, kv, 1)
    table = c["table"][:B].contiguous()
    lens, none, err = ints([20] * B), ints([0] * B), ints([0])
    p = ops.plan_step(lens, none, table, ints([1, 2]), ints([0, 2], torch.int64), page_size=16, num_blocks=c["num_blocks"],
                      num_tokens=0, error_word=err)
    assert p.total_lens.tolist() == [20] * B and p.cu_new.tolist() == [0] * (B + 1) and p.ring_pos.tolist() == [0, 2]
    rows = torch.empty(0, 2, 64, dtype=qt, device="cuda")
    if kv is I8:
        ops.append_kv_i8(rows, rows, c["k"], c["v"], c["ks"], c["vs"], block_table=table, total_lens=p.total_lens,
                         cu_new=p.cu_new, error_word=err)
    else:
        ops.append_kv(rows, rows, c["k"], c["v"], slot_map=p.slot_map, error_word=err)
    q = torch.empty(0, 8, 64, dtype=qt, device="cuda")
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], table, p.total_lens, p.cu_new, max_new=0, max_len=20, k_scale=c["ks"], v_scale=c["vs"])
    assert o.shape == q.shape
    assert a.prompt(q, rows, rows, p.cu_new, max_len=0).shape == q.shape
    assert err.item() == 0 and a.error_flag() == 0


@pytest.mark.parametrize("dt", [F16, F32])
def test_rows_of_one_head_with_any_head_stride(dt):
    """[1][tokens][dim] seen as [tokens][1][dim]: a token's values lie together whatever the stride of its one head."""
    T, D, page = 40, 64, 16
    q, k, v = (torch.empty(1, T, D, dtype=dt, device="cuda").copy_(make_q(T, 1, D, dt, s).transpose(0, 1)).transpose(0, 1)
               for s in (1, 2, 3))
    assert k.stride(1) != D
    want = attention64(q, k.double(), v.double(), 0)
    a = ops.PagedPrefill()
    assert (a.prompt(q, k, v, starts([T]), max_len=T).double() - want).abs().max().item() <= tolerance(dt)
    c = make_cache([T], [0], 1, D, page, dt, 4)
    slots = torch.arange(T, device="cuda")
    ops.append_kv(k, v, c["k"], c["v"], slot_map=c["table"][0].long()[slots // page] * page + slots % page)
    o = a.chunk(q, c["k"], c["v"], c["table"], ints([T]), starts([T]), max_new=T, max_len=T)
    assert (o.double() - want).abs().max().item() <= tolerance(dt)
    with pytest.raises(ValueError):
        a.prompt(q.expand(T, 2, D), k, v, starts([T]), max_len=T)
