"""max_new and max_len are bounds: the largest ints give the results and a workspace of ordinary size."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("kernel", [kvb.Kernel.auto, kvb.Kernel.simt])
@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("H,Hkv", [(8, 2), (4, 4), (64, 1)])
@pytest.mark.parametrize("max_new", [MOST, MOST - 1, MOST - 3, MOST - 127, MOST - 128, MOST - 255, 1 << 30, 300])
def test_chunk(kernel, qt, kv, H, Hkv, max_new):
    new, ctx = [1, 300, 0, 7], [900, 3, 5, 0]
    c = make_cache(new, ctx, Hkv, 64, 16, kv, 2)
    q = make_q(sum(new), H, 64, qt, 3)
    a = ops.PagedPrefill()
    o = a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max_new, max_len=max(max_new, 901),
                k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)
    assert a.error_flag() == 0
    at = 0
    for b, n in enumerate(new):
        if n:
            want = attention64(q[at:at + n], rows_of(c, "k", b), rows_of(c, "v", b), ctx[b])
            assert (o[at:at + n].double() - want).abs().max().item() <= tolerance(qt)
        at += n


@pytest.mark.parametrize("kernel", [kvb.Kernel.auto, kvb.Kernel.simt])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("max_len", [MOST, MOST - 60, 1 << 30])
def test_prompt(kernel, dt, max_len):
    new = [130, 1, 40]
    q, k, v = (make_q(171, h, 128, dt, h) for h in (4, 2, 3))
    v = v[:, :2].contiguous()
    a = ops.PagedPrefill()
    o = a.prompt(q, k, v, starts(new), max_len=max_len, kernel=kernel)
    assert a.error_flag() == 0
    for x, n in zip(starts(new).tolist(), new):
        y = slice(x, x + n)
        assert (o[y].double() - attention64(q[y], k[y].double(), v[y].double(), 0)).abs().max().item() <= tolerance(dt)


def test_workspace():
    K = kvb.KvType
    for tokens in (1, 1000):
        for kv, page in ((K.f16, 16), (K.i8, 128), (K.f32, 16)):
            sizes = []
            for bound in (tokens, MOST - 100, MOST):
                args = kvb.chunk_args(kvb.Shape(4, 32, 8, 128), K.f32, kv, page, 100, tokens, bound, 2 ** 20, q=0x1000,
                                      q_stride=4096, k=0x2000, v=0x3000, k_scale=0x100, v_scale=0x100, num_blocks=9,
                                      block_table=0x4000, total_lens=0x5000, cu_new=0x6000, out=0x8000, error_word=0x7000)
                sizes.append(kvb.paged_chunk_workspace_bytes(args))
            assert sizes[0] == sizes[1] == sizes[2] < 1 << 32


@pytest.mark.parametrize("bound", [2 ** 31, 2 ** 31 + 5, 2 ** 32 + 3, 2 ** 40])
def test_bounds_beyond_a_c_int(bound):
    new, ctx = [1, 30], [90, 3]
    c = make_cache(new, ctx, 2, 64, 16, F16, 2)
    q = make_q(31, 4, 64, F16, 3)
    a = ops.PagedPrefill()
    args = (q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new))
    x = a.chunk(*args, max_new=bound, max_len=bound)
    y = a.chunk(*args, max_new=2 ** 31 - 1, max_len=2 ** 31 - 1)
    assert torch.equal(x, y) and a.error_flag() == 0
    x = a.prompt(q, q[:, :2], q[:, 2:], starts(new), max_len=bound)
    assert x.isfinite().all() and a.error_flag() == 0
    for bad in (0, -1, -2 ** 32 + 50):
        with pytest.raises(ValueError):
            a.chunk(*args, max_new=bad, max_len=100)
        with pytest.raises(ValueError):
            a.prompt(q, q[:, :2], q[:, 2:], starts(new), max_len=bad)
    with pytest.raises(ValueError):
        a.chunk(*args, max_new=30, max_len=-2 ** 32 + 100)
    for page in (0, -16, 2 ** 32 + 16, 2 ** 31):
        with pytest.raises(ValueError):
            ops.plan_step(ints([0]), ints([1]), ints([[0]]), ints([0]), ints([0, 1], torch.int64), page_size=page,
                          num_blocks=1, num_tokens=1)
