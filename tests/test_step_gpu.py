"""The step plan and the append (kvb_step_plan, kvb_paged_append) on the GPU, against plain loops."""
import numpy as np
import pytest
import torch

import kv_cache_bench_b200 as kvb
from kv_cache_bench_b200 import torch_ops as ops
from tests.step_cases import F16, F32, I8, ints, make_cache, starts

pytestmark = pytest.mark.gpu


# ---- plan -------------------------------------------------------------------------------------------

def plain_plan(seq, new, table, ring, pos, page, num_blocks, T):
    table, capacity = table.copy(), table.shape[1] * page
    head, avail = pos[0], pos[1] - pos[0]
    err = 0
    if head < 0 or avail < 0 or avail > len(ring):
        err, head, avail = 8, max(head, 0), 0
    total, cu, slots, positions = [], [0], [-1] * T, [0] * T
    taken = E = at = 0
    for b, (x, n) in enumerate(zip(seq, new)):
        valid = x >= 0 and n >= 0 and x + n <= capacity
        n = max(n, 0)
        have = -(-x // page) if valid else 0
        need = -(-(x + n) // page) - have if valid else 0
        E += need
        ok = valid and at + n <= T and (need == 0 or E <= avail)
        if not valid or at + n > T:
            err |= 1
        elif not ok:
            err |= 2
        if ok and need:
            taken = E
        for i in range(n):
            if at + i >= T:
                break
            p = (x if valid else 0) + i
            positions[at + i] = p
            if not ok:
                continue
            pg = p // page
            if pg >= have:
                table[b, pg] = ring[(head + E - need + pg - have) % len(ring)]
            if 0 <= table[b, pg] < num_blocks:
                slots[at + i] = int(table[b, pg]) * page + p % page
            else:
                err |= 2
        total.append(x + n if ok else -1)
        at += n
        cu.append(min(at, T))
    return total, cu, slots, positions, [pos[0] + taken, pos[1]], table, err


def check_plan(seq, new, page, *, width=None, free=None, T=None, head=0, ring_size=None, num_blocks=None, ring=None,
               pos=None, seed=0, table=None):
    rng = np.random.default_rng(seed)
    seq, new = list(map(int, seq)), list(map(int, new))
    width = width if width is not None else max([1] + [-(-(max(x, 0) + max(n, 0)) // page) for x, n in zip(seq, new)])
    have = [min(width, -(-max(x, 0) // page)) for x in seq]
    need = sum(-(-(max(x, 0) + max(n, 0)) // page) for x, n in zip(seq, new)) - sum(have)
    free = need if free is None else free
    num_blocks = num_blocks or sum(have) + max(free, 0) + 1
    perm = rng.permutation(num_blocks).astype(np.int32)
    if table is None:
        table = np.full((len(seq), width), -7, np.int32)
        at = 0
        for b, n in enumerate(have):
            table[b, :n] = perm[at:at + n]
            at += n
    if ring is None:
        ring = np.full(ring_size or max(free, 1), -5, np.int32)
        ring[(head + np.arange(free)) % len(ring)] = perm[sum(have):sum(have) + free]
    pos = pos or [head, head + free]
    T = sum(max(n, 0) for n in new) if T is None else T
    want = plain_plan(seq, new, table, ring, pos, page, num_blocks, T)
    tb, err = ints(table), ints([0])
    p = ops.plan_step(ints(seq), ints(new), tb, ints(ring), ints(pos, torch.int64), page_size=page,
                      num_blocks=num_blocks, num_tokens=T, error_word=err)
    for got, ref in zip((p.total_lens, p.cu_new, p.slot_map, p.positions, p.ring_pos, tb, err),
                        (*want[:6], [want[6]])):
        np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(ref).reshape(got.shape))
    return p


@pytest.mark.parametrize("page", [1, 7, 16, 128])
def test_plan_matches_a_loop(page):
    rng = np.random.default_rng(page)
    for B in (1, 2, 31, 512, 513, 1300):
        seq, new = rng.integers(0, 300, B), rng.integers(0, 40, B)
        new[rng.random(B) < 0.3] = 0
        seq[rng.random(B) < 0.3] = 0
        check_plan(seq, new, page, seed=B, head=int(rng.integers(0, 1000)))


def test_plan_of_one_long_prompt_wraps_the_ring():
    check_plan([5], [100_000], 16, head=(1 << 40) + 3, ring_size=7000)


def test_plan_single_tokens_and_no_tokens():
    check_plan([0], [1], 16)
    check_plan([16], [1], 16)
    check_plan([15], [1], 16)
    check_plan([15, 3], [0, 0], 16)
    check_plan([], [], 16, width=1)
    check_plan([4, 4], [2, 2], 16, T=9)  # entries behind the last token


def test_plan_refuses_in_order_when_the_ring_runs_out():
    # the second sequence does not fit, the third would but comes later, the fourth opens no page
    p = check_plan([0, 10, 0, 3], [40, 70, 16, 5], 16, free=5)
    assert p.total_lens.tolist() == [40, -1, -1, 8]
    assert p.ring_pos.tolist() == [3, 5]


def test_plan_refuses_bad_lengths_and_capacity():
    check_plan([-1, 4, 4, 0], [3, -2, 100, 6], 16, width=3)
    check_plan([2 ** 31 - 1, 4], [2 ** 31 - 1, 3], 16, width=3, T=8, free=4)  # sums that pass 32 bits
    check_plan([4, 4, 4], [8, 8, 8], 16, T=17)


def test_plan_reports_bad_ids_and_a_bad_ring():
    check_plan([0, 0], [20, 20], 16, ring=np.array([0, 99, -3, 1], np.int32), pos=[0, 4], num_blocks=4)
    check_plan([20], [3], 16, table=np.array([[1, 77]], np.int32), num_blocks=4, free=0)
    for pos in ([-1, 2], [3, 2], [0, 9]):
        check_plan([3, 0], [2, 5], 16, pos=pos, ring=np.arange(4, dtype=np.int32), num_blocks=8,
                   table=np.array([[6], [-7]], np.int32))


def test_pages_go_round():
    """Requests come and go for many steps on a small ring: no live page is ever handed out twice, and every
    page comes back."""
    rng = np.random.default_rng(0)
    B, page, num_blocks, width = 5, 4, 30, 9
    ring = ints(rng.permutation(num_blocks))
    pos = ints([0, num_blocks], torch.int64)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    lens, err = ints([0] * B), ints([0])
    for step in range(60):
        room = width * page - lens.cpu().numpy()
        new = np.minimum(rng.integers(0, 9, B), room)
        p = ops.plan_step(lens, ints(new), table, ring, pos, page_size=page, num_blocks=num_blocks,
                          num_tokens=int(new.sum()), error_word=err)
        lens, pos = torch.where(p.total_lens < 0, lens, p.total_lens), p.ring_pos
        b = int(rng.integers(0, B))
        if rng.random() < 0.5:  # request b ends
            pages = -(-int(lens[b]) // page)
            ring[(pos[1] + torch.arange(pages, device="cuda")) % num_blocks] = table[b, :pages]
            pos[1] += pages
            lens[b] = 0
        owned = [table[i, j].item() for i in range(B) for j in range(-(-int(lens[i]) // page))]
        head, tail = pos.tolist()
        free = ring[torch.arange(head, tail, device="cuda") % num_blocks].tolist()
        assert sorted(owned + free) == list(range(num_blocks)), step
    assert pos[0].item() > num_blocks and err.item() in (0, 2)


# ---- append -----------------------------------------------------------------------------------------

def source(T, Hkv, D, dtype, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.full((T, Hkv * D + pad), float("nan"), dtype=dtype, device="cuda")
    y = torch.empty(T, Hkv * D, device="cuda").uniform_(-1, 1, generator=g)
    y *= torch.exp2(-torch.randint(0, 6, (T, 1), device="cuda", generator=g).float())
    x[:, :Hkv * D] = y.to(dtype)
    return x[:, :Hkv * D].view(T, Hkv, D)


def slots_of(c, new, ctx):
    out = [int(c["table"][b, p // c["page"]]) * c["page"] + p % c["page"]
           for b, (n, x) in enumerate(zip(new, ctx)) for p in range(x, x + n)]
    return ints(out, torch.int64)


STEPS = [([1], [0]), ([1, 1, 1], [15, 16, 17]), ([37, 0, 1, 130], [5, 9, 0, 64]), ([300], [0])]


@pytest.mark.parametrize("src,kv", [(F16, F16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("Hkv,D,page", [(8, 128, 16), (1, 64, 7), (3, 72, 128)])
def test_append_rows(src, kv, Hkv, D, page):
    for i, (new, ctx) in enumerate(STEPS):
        c = make_cache(new, ctx, Hkv, D, page, kv, seed=i)
        T = sum(new)
        k, v = source(T, Hkv, D, src, i, pad=8), source(T, Hkv, D, src, i + 50)
        slots = slots_of(c, new, ctx)
        if T > 2:
            slots[1] = -1
        want = []
        for x, rows in (("k", k), ("v", v)):
            w = c[x].clone()
            for t, s in enumerate(slots.tolist()):
                if s >= 0:
                    w[s // page, :, s % page] = rows[t].to(kv)
            want.append(w)
        err = ints([0])
        ops.append_kv(k, v, c["k"], c["v"], slot_map=slots, error_word=err)
        for got, w in zip((c["k"], c["v"]), want):
            assert torch.equal(got.view(torch.int16 if kv is F16 else torch.int32),
                               w.view(torch.int16 if kv is F16 else torch.int32))
        assert err.item() == 0


def test_append_rows_skips_bad_slots():
    c = make_cache([4], [0], 2, 64, 16, F16, seed=1)
    k = source(4, 2, 64, F16, 1)
    before, err = c["k"].clone(), ints([0])
    ops.append_kv(k, k, c["k"], c["v"], slot_map=ints([-2, c["num_blocks"] * 16, 1 << 40, -1], torch.int64), error_word=err)
    assert err.item() == 2 and torch.equal(c["k"].view(torch.int16), before.view(torch.int16))


def plain_append_i8(pool, scale, rows, c, new, ctx):
    """The rule in fp32 operations, one page and head at a time, in numpy (IEEE division, ties to even)."""
    pool, scale, rows = pool.cpu().numpy().copy(), scale.cpu().numpy().copy(), rows.float().cpu().numpy()
    table, page, t = c["table"].cpu().numpy(), c["page"], 0
    for b, (n, x) in enumerate(zip(new, ctx)):
        p = x
        while p < x + n:
            blk, r0 = table[b, p // page], p % page
            m = min(page - r0, x + n - p)
            for h in range(rows.shape[1]):
                y = rows[t:t + m, h]
                s = np.float32(np.abs(y).max()) / np.float32(127)
                if r0:
                    old = scale[blk, h]
                    if old >= s:
                        s = old
                    else:
                        ratio = np.float32(old) / s
                        pool[blk, h, :r0] = np.rint(pool[blk, h, :r0].astype(np.float32) * ratio)
                scale[blk, h] = s
                q = np.zeros_like(y) if s == 0 else np.clip(np.rint(y / s), -127, 127)
                pool[blk, h, r0:r0 + m] = q
            p, t = p + m, t + m
    return pool, scale


@pytest.mark.parametrize("src", [F16, F32])
@pytest.mark.parametrize("Hkv,D,page", [(8, 128, 16), (1, 64, 7), (3, 72, 128)])
def test_append_i8(src, Hkv, D, page):
    for i, (new, ctx) in enumerate(STEPS + [([1] * 70, list(range(70))), ([60] * 40, list(range(40)))]):
        c = make_cache(new, ctx, Hkv, D, page, I8, seed=i)
        T = sum(new)
        k, v = source(T, Hkv, D, src, i, pad=8), source(T, Hkv, D, src, i + 50)
        if T > 30:
            k[3:] *= 0.0  # pages of zeros
        want = [plain_append_i8(c[x], c[x + "s"], r, c, new, ctx) for x, r in (("k", k), ("v", v))]
        err = ints([0])
        ops.append_kv_i8(k, v, c["k"], c["v"], c["ks"], c["vs"], block_table=c["table"], total_lens=ints(c["total"]),
                         cu_new=starts(new), error_word=err)
        for x, (pool, scale) in zip("kv", want):
            np.testing.assert_array_equal(c[x].cpu().numpy(), pool)
            np.testing.assert_array_equal(c[x + "s"].cpu().numpy(), scale)
        assert err.item() == 0


def test_append_i8_of_whole_prompts_is_the_page_quantizer():
    new, Hkv, D, page = [100, 33, 128], 4, 128, 32
    c = make_cache(new, [0] * 3, Hkv, D, page, I8, seed=3)
    k = source(sum(new), Hkv, D, F32, 5)
    ref, refs = c["k"].clone(), c["ks"].clone()
    contig = torch.zeros(3, Hkv, max(new), D, device="cuda")
    for b, (a, n) in enumerate(zip(starts(new).tolist(), new)):
        contig[b, :, :n] = k[a:a + n].transpose(0, 1)
    lens = ints(new)
    kvb.quantize_paged_i8(kvb.page_write_args(3, Hkv, D, kvb.KvType.i8, page, c["table"].shape[1], max(new),
                                              contig=contig.data_ptr(), block_table=c["table"].data_ptr(),
                                              seq_lens=lens.data_ptr(), pool=ref.data_ptr(),
                                              num_blocks=c["num_blocks"], scales=refs.data_ptr()),
                          torch.cuda.current_stream().cuda_stream)
    ops.append_kv_i8(k, k, c["k"], c["v"], c["ks"], c["vs"], block_table=c["table"], total_lens=lens, cu_new=starts(new))
    assert torch.equal(c["k"], ref)
    assert torch.equal(c["ks"].nan_to_num(-1), refs.nan_to_num(-1))


def test_append_i8_skips_refused_sequences():
    new, ctx = [4, 4, 4, 4], [0, 20, 0, 3]
    c = make_cache(new, ctx, 2, 64, 16, I8, seed=8)
    k = source(16, 2, 64, F16, 1)
    total = ints([-1, 3, 4, 10_000])  # refused by the plan; below its new tokens; served; beyond the table
    c["table"][2, 0] = c["num_blocks"]  # ... but its page is outside the pool
    before, err = c["k"].clone(), ints([0])
    ops.append_kv_i8(k, k, c["k"], c["v"], c["ks"], c["vs"], block_table=c["table"], total_lens=total,
                     cu_new=starts(new), error_word=err)
    assert err.item() == 3 and torch.equal(c["k"], before)
    err.zero_()
    ops.append_kv_i8(k[:4], k[:4], c["k"], c["v"], c["ks"], c["vs"], block_table=c["table"][:1].contiguous(),
                     total_lens=ints([-1]), cu_new=starts([4]), error_word=err)
    assert err.item() == 0 and torch.equal(c["k"], before)


def test_tensors_are_checked():
    c = make_cache([4], [0], 2, 64, 16, F16, seed=1)
    k = source(4, 2, 64, F16, 1)
    slots = ints([0, 1, 2, 3], torch.int64)
    for bad in (dict(slot_map=slots.int()), dict(slot_map=slots[:3]), dict(slot_map=slots.cpu()),
                dict(slot_map=slots, error_word=torch.zeros(1, device="cuda"))):
        with pytest.raises(ValueError):
            ops.append_kv(k, k, c["k"], c["v"], **bad)
    with pytest.raises(ValueError):
        ops.append_kv(k.transpose(0, 1), k.transpose(0, 1), c["k"], c["v"], slot_map=slots)
    with pytest.raises(ValueError):
        ops.append_kv(k, k, c["k"].char(), c["v"].char(), slot_map=slots)
    with pytest.raises(ValueError):
        ops.plan_step(ints([0]), ints([1]).long(), ints([[0]]), ints([0]), ints([0, 1], torch.int64), page_size=16,
                      num_blocks=1, num_tokens=1)
