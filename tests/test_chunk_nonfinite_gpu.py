"""Non-finite values and keys in attention of several new tokens per sequence, in units of one and of two
query tiles, whole and cut: they reach the tokens that see them, and no other."""
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, attention64, ints, make_cache, make_q, rows_of, starts, tolerance

pytestmark = pytest.mark.gpu
AUTO, SIMT = kvb.Kernel.auto, kvb.Kernel.simt


def same(o, want, qt):
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(o))
    assert torch.where(fine, o.double() - want, 0.0).abs().max().item() <= tolerance(qt)


# Query heads per KV head, new tokens, tokens before them, and where the values lie: before the unit's second
# query tile, with the tiles' first masked key tiles the same and different ones.
PLACES = [(1, 256, 0, 5), (1, 256, 0, 127), (1, 256, 0, 128), (1, 600, 0, 300), (1, 200, 60, 70), (4, 64, 100, 110),
          (4, 40, 100, 127), (4, 64, 100, 128), (4, 64, 3000, 3010), (2, 500, 2000, 2100), (7, 36, 120, 122),
          (64, 4, 126, 127)]


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,n,ctx,at", PLACES)
def test_values_of_the_new_tokens(kernel, qt, kv, D, G, n, ctx, at):
    c = make_cache([n], [ctx], 2, D, 16, kv, seed=5)
    q = make_q(n, 2 * G, D, qt, 6)
    for d, (p, x) in enumerate(((at, float("inf")), (at + 1, float("nan")), (at + 2, -float("inf")))):
        if p < n + ctx:
            c["v"][c["table"][0, p // 16].long(), 0, p % 16, 3 + d] = x
    o = ops.PagedPrefill().chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts([n]), max_new=n, max_len=n + ctx,
                                 kernel=kernel)
    same(o, attention64(q, rows_of(c, "k", 0), rows_of(c, "v", 0), ctx), qt)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("G,n,at", [(G, n, at) for G, n, ctx, at in PLACES if ctx == 0] + [(4, 3000, 1030)])
def test_values_of_a_prompt(kernel, dt, G, n, at):
    q, k, v = (make_q(n + 9, h, 128, dt, h) for h in (2 * G, 2, 3))
    v = v[:, :2].contiguous()
    v[at, 0, 3], v[at + 1, 0, 4], v[at + 2, 0, 5] = float("inf"), float("nan"), -float("inf")
    o = ops.PagedPrefill().prompt(q, k, v, starts([n, 9]), max_len=n, kernel=kernel)
    for x in (slice(0, n), slice(n, n + 9)):
        same(o[x], attention64(q[x], k[x].double(), v[x].double(), 0), dt)


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,n,ctx,at", [(4, 40, 100, [3]), (1, 300, 0, [0, 70, 200]), (4, 5, 3000, [10, 31, 32, 1500, 3001]),
                                        (2, 200, 700, list(range(50, 600, 7))), (8, 3, 200, list(range(128)))])
def test_infinite_keys(kernel, qt, kv, D, G, n, ctx, at):
    """An infinite component of a key scores -inf (no weight) or +inf (NaN) by the query's sign, and NaN where that is
    0 or another component is infinite the other way; queries too small for the fp16 parts of the row count too."""
    c = make_cache([n], [ctx], 2, D, 16, kv, seed=5)
    q = make_q(n, 2 * G, D, qt, 6)
    q[:, :, 7] = -q[:, :, 7].abs() - 0.25
    q[:, 1:, 9] = q[:, 1:, 9].abs() + 1e-3  # (head 0: any sign)
    q[n // 2, 0, 9] = 0.0
    if qt is F32:
        q[1::3, :, 7] = -1e-9
        q[n - 1, -1, 7] = -1e-30
    for i, p in enumerate(at):
        k = c["k"][c["table"][0, p // 16].long()]
        k[0, p % 16, 7 if i % 2 == 0 else 9] = float("inf") if i % 2 == 0 else -float("inf")
        k[1, p % 16, 7] = float("inf")
        if i == 2:
            k[1, p % 16, 9] = -float("inf")
    a = ops.PagedPrefill()

    def run():
        return a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts([n]), max_new=n, max_len=n + ctx,
                       kernel=kernel)

    o = run()
    want = attention64(q, rows_of(c, "k", 0), rows_of(c, "v", 0), ctx)
    assert want[:, 2 * G - 1].isfinite().any()
    same(o, want, qt)
    assert torch.equal(o.nan_to_num(7), run().nan_to_num(7))


@pytest.mark.parametrize("kernel", [AUTO, SIMT])
@pytest.mark.parametrize("qt,kv", [(F16, F16), (F32, F16), (F16, I8), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("new,ctx", [([150], [100]), ([3, 40], [3000, 0])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_queries_stay_in_their_rows(kernel, qt, kv, new, ctx, bad):
    c = make_cache(new, ctx, 2, 128, 16, kv, seed=5)
    q = make_q(sum(new), 8, 128, qt, 6)
    a = ops.PagedPrefill()

    def run():
        return a.chunk(q, c["k"], c["v"], c["table"], ints(c["total"]), starts(new), max_new=max(new),
                       max_len=max(c["total"]), k_scale=c["ks"], v_scale=c["vs"], kernel=kernel)

    want = run().double()
    rows = torch.zeros(sum(new), 8, dtype=torch.bool, device="cuda")
    rows[::3, 1] = rows[1, 5] = rows[sum(new) - 1, 7] = True
    q[rows] = torch.where(torch.arange(128, device="cuda") == 77, bad, q[rows])
    o = run()
    assert o[rows].isnan().all()  # (an infinite component scores +inf against some key, and NaN follows)
    assert (o[~rows].double() - want[~rows]).abs().max().item() <= 2 * tolerance(qt)
