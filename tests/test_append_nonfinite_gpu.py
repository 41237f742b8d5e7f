"""Rows that are not finite in the append into int8 pages: their page's scale says so, whatever lies beside
them, until the page is begun anew."""
import numpy as np
import pytest
import torch

from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, ints, make_cache, starts
from tests.test_step_gpu import plain_append_i8, source

pytestmark = pytest.mark.gpu


def append(c, k, v, new):
    err = ints([0])
    ops.append_kv_i8(k, v, c["k"], c["v"], c["ks"], c["vs"], block_table=c["table"], total_lens=ints(c["total"]),
                     cu_new=starts(new), error_word=err)
    assert err.item() == 0


@pytest.mark.parametrize("src", [F16, F32])
@pytest.mark.parametrize("Hkv,D,page", [(2, 128, 16), (1, 64, 7), (3, 72, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,ctx", [([300, 40], [0, 20]), ([1, 1, 1], [0, 5, 17])])
def test_a_nonfinite_row_marks_its_pages_scale(src, Hkv, D, page, bad, new, ctx):
    c = make_cache(new, ctx, Hkv, D, page, I8, seed=2)
    k, v = source(sum(new), Hkv, D, src, 3), source(sum(new), Hkv, D, src, 4)
    want, touched = {}, set()
    cu = starts(new).tolist()
    for x, rows in (("k", k), ("v", v)):
        want[x] = plain_append_i8(c[x], c[x + "s"], rows, c, new, ctx)
    for b, i, h in ((0, 0, 0), (0, 40, Hkv - 1), (1, 0, Hkv - 1), (1, 33, 0)):
        if i < new[b]:
            k[cu[b] + i, h, 5 * i % D] = bad
            touched.add((int(c["table"][b, (ctx[b] + i) // page]), h))
    append(c, k, v, new)
    marked = torch.zeros_like(c["ks"], dtype=torch.bool)
    for blk, h in touched:
        marked[blk, h] = True
    assert (c["ks"][marked].isnan() if bad != bad else c["ks"][marked].isinf()).all()
    live = torch.zeros(c["num_blocks"], dtype=torch.bool, device="cuda")
    for b, t in enumerate(c["total"]):
        live[c["table"][b, :-(-t // page)].long()] = True
    values = c["k"].float() * c["ks"][:, :, None, None]
    for blk, h in touched:
        assert values[blk, h].isnan().logical_or(values[blk, h].isinf()).all()
    keep = ~marked.cpu().numpy()
    np.testing.assert_array_equal(c["k"].cpu().numpy()[keep], want["k"][0][keep])
    np.testing.assert_array_equal(c["ks"].cpu().numpy()[keep], want["k"][1][keep])
    np.testing.assert_array_equal(c["v"].cpu().numpy(), want["v"][0])


@pytest.mark.parametrize("D,page", [(64, 16), (128, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_the_mark_stays_until_the_page_is_begun_anew(D, page, bad):
    c = make_cache([page], [0], 2, D, page, I8, seed=2)
    k = source(page, 2, D, F32, 3)
    k[3, 1, 9] = bad
    for n in range(0, page, 8):  # eight tokens at a time
        c["total"] = [n + 8]
        append(c, k[n:n + 8], k[n:n + 8], [8])
        blk = c["table"][0, 0].long()
        for s in (c["ks"][blk], c["vs"][blk]):
            assert s[0].isfinite() and not s[1].isfinite()
    rows = source(page, 2, D, F32, 5)
    c["total"] = [page]
    append(c, rows, rows, [page])
    assert c["ks"][blk].isfinite().all()
    assert (c["k"][blk].float() * c["ks"][blk][:, None, None] - rows.transpose(0, 1)).abs().max() <= 1 / 253
