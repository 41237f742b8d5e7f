"""The cases of the operators that a serving step of several tokens needs beside single-token decode:
planning the step's pages (`plan_step`), writing its keys and values into the paged cache
(`append_kv`), attention of the new tokens over that cache (`PagedPrefill.chunk`) and causal
attention over whole packed prompts (`PagedPrefill.prompt`).

`run` computes each in plain torch operations, or, with `own` set, calls the framework. Head layouts
(32 or 64 query heads over 8 KV heads, head dims 64 and 128), page sizes (16 to 128) and context
lengths (512 to 131072 tokens) are those of the framework's decode configurations.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "i8": 1}


# ---- cases --------------------------------------------------------------------------------------

def _case(name, op, **kw):
    c = dict(op=op, batch=1, heads=32, kv_heads=8, dim=128, page=16, new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=0,
             src="f16", kv="f16", lens=1)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of a serving batch: every sequence gets one token, a few open a new page
        _case("plan_decode_256", "plan", batch=256, page=64, ctx_lo=8192, ctx_hi=131072, lens=11),
        # a step that admits ragged prompts (the lengths of the 64-sequence configuration, page 16)
        _case("plan_prompts_64", "plan", batch=64, page=16, new_lo=512, new_hi=32768, lens=12),
        # the decode step's own token of 64 sequences into fp16 pages: latency counts
        _case("append_decode_f16", "append", batch=64, page=16, ctx_lo=512, ctx_hi=4096, lens=13),
        # prompts of ordinary length quantized into int8 pages of 128 tokens, from fp32 projections
        _case("append_prompt_i8", "append", batch=3, page=128, new_lo=512, new_hi=4096, ctx_lo=1, ctx_hi=512,
              src="f32", kv="i8", lens=14),
        # a long admitted batch into fp16 pages, keys and values in fp32 as the decode path's queries are
        _case("append_prompt_f16", "append", batch=16, page=32, new_lo=512, new_hi=4096, ctx_lo=0, ctx_hi=300,
              src="f32", kv="f16", lens=15),
        # a few drafted tokens verified over a 4 k context: one query tile a sequence, latency counts
        _case("chunk_verify_f16", "chunk", batch=4, page=32, new_lo=3, new_hi=8, ctx_lo=3000, ctx_hi=4096, lens=16),
        # chunked prefill of the 32 k int8 configuration, fp32 queries as its decode step has
        _case("chunk_512_of_32k_i8", "chunk", batch=1, page=128, new_lo=512, new_hi=512, ctx_lo=32256, ctx_hi=32256,
              src="f32", kv="i8", lens=17),
        # a ragged batch: some sequences continue a prompt, some have only a few tokens
        _case("chunk_ragged_f16", "chunk", batch=8, page=16, new_lo=1, new_hi=256, ctx_lo=512, ctx_hi=30000, lens=18),
        # a large chunk on a long context
        _case("chunk_2048_of_32k_f16", "chunk", batch=1, page=64, new_lo=2048, new_hi=2048, ctx_lo=30720,
              ctx_hi=30720, lens=19),
        # the 512-token fp32 configuration, a chunk of 61 tokens
        _case("chunk_f32", "chunk", batch=2, page=16, new_lo=61, new_hi=61, ctx_lo=451, ctx_hi=451, src="f32",
              kv="f32", lens=20),
        # one whole prompt
        _case("prompt_8192_f16", "prompt", batch=1, new_lo=8192, new_hi=8192, lens=21),
        # packed prompts of odd lengths
        _case("prompt_ragged_f16", "prompt", batch=12, heads=64, new_lo=33, new_hi=2500, lens=22),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "chunk", "prompt"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (8, 2), (16, 16), (12, 4), (40, 8), (7, 1)])
    c = _case(None, op, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]),
              page=rng.choice([16, 32, 64, 128]), lens=rng.randrange(1 << 30))
    if op == "plan":
        c.update(batch=_log_int(rng, 1, 1024), new_hi=_log_int(rng, 1, 4096), ctx_hi=_log_int(rng, 1, 8192))
        if c["batch"] * c["new_hi"] > 1 << 20:
            c["new_hi"] = (1 << 20) // c["batch"]
    elif op == "append":
        c.update(batch=_log_int(rng, 1, 128), new_hi=_log_int(rng, 1, 4096), ctx_hi=_log_int(rng, 1, 2048),
                 kv=rng.choice(["f16", "f16", "i8", "f32"]))
        c["src"] = "f32" if c["kv"] == "f32" else rng.choice(["f16", "f32"])
        if c["batch"] * c["new_hi"] > 16384:
            c["new_hi"] = 16384 // c["batch"]
    elif op == "chunk":
        c.update(batch=_log_int(rng, 1, 16), new_hi=_log_int(rng, 1, 2048), ctx_hi=_log_int(rng, 64, 32768),
                 kv=rng.choice(["f16", "f16", "i8", "i8", "f32"]))
        c["src"] = "f32" if c["kv"] == "f32" else rng.choice(["f16", "f32"])
        most = (1 << 29) if c["kv"] != "f32" else (1 << 25)  # query-key pairs times heads
        while c["batch"] * heads * c["new_hi"] * (c["new_hi"] + c["ctx_hi"]) > most:
            c["new_hi"], c["ctx_hi"] = max(1, c["new_hi"] * 3 // 4), max(1, c["ctx_hi"] * 3 // 4)
    else:
        c.update(batch=_log_int(rng, 1, 32), new_hi=_log_int(rng, 1, 8192), src=rng.choice(["f16", "f16", "f32"]))
        c["kv"] = c["src"]
        most = (1 << 29) if c["kv"] != "f32" else (1 << 25)
        while c["batch"] * heads * c["new_hi"] ** 2 > most:
            c["new_hi"] = max(1, c["new_hi"] * 3 // 4)
    c["new_lo"] = 1
    return c


def _lens(c):
    """The sequences' new tokens and the tokens cached before them: whole numbers, spread over their
    logarithm, the same for every seed."""
    rng = random.Random(c["lens"])
    new = [_log_int(rng, c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
    ctx = [_log_int(rng, c["ctx_lo"] + 1, c["ctx_hi"] + 1) - 1 for _ in range(c["batch"])]
    return new, ctx


def _up(x, page):
    return (x + page - 1) // page


def work(c):
    new, ctx = _lens(c)
    T, row = sum(new), c["kv_heads"] * c["dim"]
    if c["op"] == "plan":
        # lengths, the lengths after the step, the starts; slots and positions; the new pages' ids read
        # from the ring and written to the table, and the id of a page that was open already
        pages = sum(_up(x + n, c["page"]) - _up(x, c["page"]) for n, x in zip(new, ctx))
        return {"bytes": 16 * c["batch"] + 12 * T + 8 * pages + 4 * c["batch"], "flops": 0}
    if c["op"] == "append":
        scales = 16 * c["kv_heads"] * sum(_up(x + n, c["page"]) - x // c["page"] for n, x in zip(new, ctx))
        return {"bytes": 2 * T * row * (BYTES[c["src"]] + BYTES[c["kv"]]) + (scales if c["kv"] == "i8" else 8 * T),
                "flops": 0}
    pairs = sum(n * x + n * (n + 1) // 2 for n, x in zip(new, ctx)) if c["op"] == "chunk" else \
        sum(n * (n + 1) // 2 for n in new)
    keys = sum(new) + (sum(ctx) if c["op"] == "chunk" else 0)
    return {"bytes": 2 * T * c["heads"] * c["dim"] * BYTES[c["src"]] + 2 * keys * row * BYTES[c["kv"]],
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- inputs -------------------------------------------------------------------------------------

def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + c["lens"])
    new, ctx = _lens(c)
    B, T, Hkv, D, page = c["batch"], sum(new), c["kv_heads"], c["dim"], c["page"]
    total = [n + x for n, x in zip(new, ctx)]
    s = dict(case=c, T=T, page=page, max_new=max(new), max_len=max(total), kept={})
    s["new_lens"], s["seq_lens"], s["total_lens"] = _ints(new), _ints(ctx), _ints(total)
    s["cu_new"] = _ints([0] + torch.tensor(new).cumsum(0).tolist())

    def rand(*shape, dtype):
        x = torch.empty(shape, dtype=torch.float32, device="cuda")
        return x.normal_(generator=g).to(DTYPES[dtype])

    if c["op"] == "prompt":
        # one fused projection's output, as a model has it: q, k and v are its column ranges
        H = c["heads"]
        qkv = rand(T, (H + 2 * Hkv) * D, dtype=c["src"])
        s["q"], s["k"], s["v"] = (qkv[:, a * D:b * D].view(T, b - a, D)
                                  for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
        return s

    # a shuffled pool with a tenth of slack: every sequence's pages, and the free ids in a ring
    pages = [_up(x, page) for x in (ctx if c["op"] == "plan" else total)]
    num_blocks = int(1.1 * sum(_up(x, page) for x in total)) + 2
    perm = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
    width = max(_up(x, page) for x in total) + 1
    used = torch.arange(width, device="cuda")[None, :] < _ints(pages)[:, None]
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[used] = perm[:sum(pages)]
    s["block_table"], s["num_blocks"] = table, num_blocks
    if c["op"] == "plan":
        free = perm[sum(pages):]
        head = int(torch.randint(0, 1 << 20, (1,), generator=g, device="cuda"))
        s["ring"] = torch.full((num_blocks,), -1, dtype=torch.int32, device="cuda")
        s["ring"][(head + torch.arange(free.numel(), device="cuda")) % num_blocks] = free
        s["ring_pos"] = _ints([head, head + free.numel()], torch.int64)
        return s

    # pages as earlier steps left them: live values, and stale ones behind the last token
    shape = (num_blocks, Hkv, page, D)
    if c["kv"] == "i8":
        for x in "kv":
            s[x + "_pool"] = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=g)
            s[x + "_scale"] = torch.empty(num_blocks, Hkv, device="cuda").uniform_(0.015, 0.035, generator=g)
    else:
        for x in "kv":
            s[x + "_pool"] = torch.empty(shape, dtype=DTYPES[c["kv"]], device="cuda")
            for piece in s[x + "_pool"].split(max(1, (1 << 27) // (Hkv * page * D))):
                piece.copy_(torch.empty(piece.shape, device="cuda").normal_(generator=g))
    if c["op"] == "append":
        kv = rand(T, 2 * Hkv * D, dtype=c["src"])
        s["k"], s["v"] = kv[:, :Hkv * D].view(T, Hkv, D), kv[:, Hkv * D:].view(T, Hkv, D)
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), s["new_lens"].long())
        pos = torch.arange(T, device="cuda") - s["cu_new"][seq] + s["seq_lens"][seq]
        s["slot_map"] = table[seq, pos // page].long() * page + pos % page
    else:
        s["q"] = rand(T, c["heads"], D, dtype=c["src"])
    return s


# ---- the plain forms ----------------------------------------------------------------------------

def _token_places(s, cu_new, seq_lens):
    """Each token's sequence and its position in it."""
    t = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(cu_new[1:].contiguous(), t, right=True)
    return seq, t - cu_new[seq] + seq_lens[seq]


def _plan(s):
    page, table, ring = s["page"], s["block_table"], s["ring"]
    seq_lens, new_lens = s["seq_lens"].long(), s["new_lens"].long()
    total = seq_lens + new_lens
    cu = torch.cat([new_lens.new_zeros(1), new_lens.cumsum(0)])
    have = (seq_lens + page - 1) // page
    need = (total + page - 1) // page - have
    ends = need.cumsum(0)
    fits = (need == 0) | (ends <= s["ring_pos"][1] - s["ring_pos"][0])
    head = s["ring_pos"][:1] + torch.where(fits, ends, 0).amax()
    seq, pos = _token_places(s, cu, seq_lens)
    lp = pos // page
    fresh = s["ring_pos"][0] + ends[seq] - need[seq] + lp - have[seq]
    block = torch.where(lp < have[seq], table[seq, lp], ring[fresh % ring.numel()])
    opens = (lp >= have[seq]) & fits[seq]
    table[seq, lp] = torch.where(opens, block, table[seq, lp])
    slots = torch.where(fits[seq], block.long() * page + pos % page, -1)
    total = torch.where(fits, total, -1).int()
    return total, cu.int(), slots, pos.int(), torch.cat([head, s["ring_pos"][1:]]), table


def _append_rows(pool, rows, slots):
    num_blocks, Hkv, page, D = pool.shape
    pool.transpose(1, 2)[slots // page, slots % page] = rows.to(pool.dtype)
    return pool


def _append_i8(s, rows, pool, scale):
    num_blocks, Hkv, page, D = pool.shape
    rows = rows.float()
    block, at = s["slot_map"] // page, s["slot_map"] % page
    amax = torch.zeros_like(scale).index_reduce_(0, block, rows.abs().amax(2), "amax")
    first = torch.full((num_blocks,), page, dtype=torch.long, device="cuda").index_reduce_(0, block, at, "amin")
    new = amax / torch.full_like(amax, 127.0)  # a true division: by a number it would be a product with 1 / 127
    kept = torch.where((first > 0)[:, None], scale, 0.0)  # a page that starts with this step has no scale yet
    new = torch.where((first == page)[:, None], scale, torch.maximum(kept, new))
    grown = ((first > 0) & (first < page))[:, None] & (new > kept)
    ratio = torch.where(grown, kept / new, 1.0)
    old = torch.arange(page, device="cuda")[None, :] < first[:, None]
    again = torch.round(pool.float() * ratio[:, :, None, None])
    pool.copy_(torch.where(old[:, None, :, None], again, pool.float()))
    per = new[block][:, :, None]
    q = torch.where(per > 0, torch.round(rows / per), 0.0).clamp(-127, 127)
    pool.transpose(1, 2)[block, at] = q.to(torch.int8)
    scale.copy_(new)


def _values(pool, scale):
    """What an int8 pool stands for."""
    return pool.float() * scale[:, :, None, None]


def _append(s):
    if s["case"]["kv"] != "i8":
        return _append_rows(s["k_pool"], s["k"], s["slot_map"]), _append_rows(s["v_pool"], s["v"], s["slot_map"])
    _append_i8(s, s["k"], s["k_pool"], s["k_scale"])
    _append_i8(s, s["v"], s["v_pool"], s["v_scale"])
    return _append_values(s)


def _append_values(s):
    return _values(s["k_pool"], s["k_scale"]), _values(s["v_pool"], s["v_scale"]), s["k_scale"], s["v_scale"]


def _attend(q, k, v, cu_new, ctx, max_new):
    """Causal attention of padded sequences: q packed [T][H][D], k and v [B][L][Hkv][D] in 32 bits,
    sequence b's first new token at position ctx[b]."""
    T, H, D = q.shape
    B, L, Hkv, _ = k.shape
    cu = cu_new.long()
    i = torch.arange(max_new, device="cuda")
    rows = (cu[:B, None] + i).clamp(max=T - 1)
    qp = q[rows].float().view(B, max_new, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    sc = (qp @ k.permute(0, 2, 3, 1)).view(B, Hkv, H // Hkv, max_new, L)
    sc *= 1.0 / math.sqrt(D)
    seen = torch.arange(L, device="cuda")[None, None, :] <= (ctx.long()[:, None] + i)[:, :, None]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    sc -= sc.amax(-1, keepdim=True)
    sc.exp_()
    sums = sc.sum(-1)
    o = (sc.view(B, Hkv, -1, L) @ v.transpose(1, 2)).view(B, Hkv, H // Hkv, max_new, D) / sums[..., None]
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, max_new, H, D)[seq, t - cu[seq]].to(q.dtype)


def _chunk(s):
    def gathered(pool, scale):
        n = _up(s["max_len"], s["page"])
        ids = s["block_table"][:, :n].clamp(min=0).long()
        x = pool[ids].float()
        if scale is not None:
            x = x * scale[ids][..., None, None]
        x = x.transpose(2, 3).reshape(ids.shape[0], n * s["page"], pool.shape[1], pool.shape[3])[:, :s["max_len"]]
        live = torch.arange(s["max_len"], device="cuda")[None, :] < s["total_lens"][:, None]
        return torch.where(live[:, :, None, None], x, 0.0)

    k, v = gathered(s["k_pool"], s.get("k_scale")), gathered(s["v_pool"], s.get("v_scale"))
    return _attend(s["q"], k, v, s["cu_new"], s["seq_lens"], s["max_new"])


def _prompt(s):
    cu = s["cu_new"].long()
    i = torch.arange(s["max_new"], device="cuda")
    rows = (cu[:-1, None] + i).clamp(max=s["T"] - 1)
    return _attend(s["q"], s["k"][rows].float(), s["v"][rows].float(), cu, torch.zeros_like(s["seq_lens"]),
                   s["max_new"])


def run(s):
    op = s["case"]["op"]
    if own:
        from kv_cache_bench_b200 import torch_ops as ops

        if op == "plan":
            p = ops.plan_step(s["seq_lens"], s["new_lens"], s["block_table"], s["ring"], s["ring_pos"],
                              page_size=s["page"], num_blocks=s["num_blocks"], num_tokens=s["T"])
            return p.total_lens, p.cu_new, p.slot_map, p.positions, p.ring_pos, s["block_table"]
        if op == "append":
            if s["case"]["kv"] != "i8":
                ops.append_kv(s["k"], s["v"], s["k_pool"], s["v_pool"], slot_map=s["slot_map"])
                return s["k_pool"], s["v_pool"]
            ops.append_kv_i8(s["k"], s["v"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"],
                             block_table=s["block_table"], total_lens=s["total_lens"], cu_new=s["cu_new"])
            return _append_values(s)
        if "attention" not in s["kept"]:
            s["kept"]["attention"] = ops.PagedPrefill()  # holds the workspace from call to call
        attention = s["kept"]["attention"]
        if op == "chunk":
            return attention.chunk(s["q"], s["k_pool"], s["v_pool"], s["block_table"], s["total_lens"], s["cu_new"],
                                   max_new=s["max_new"], max_len=s["max_len"], k_scale=s.get("k_scale"),
                                   v_scale=s.get("v_scale"))
        return attention.prompt(s["q"], s["k"], s["v"], s["cu_new"], max_len=s["max_new"])
    return {"plan": _plan, "append": _append, "chunk": _chunk, "prompt": _prompt}[op](s)


# ---- in 64 bits -----------------------------------------------------------------------------------

def exact(c, seed):
    def attention(q, keys, values, first):
        # one sequence: q [n][H][D], keys and values [L][Hkv][D] in float64, query i at position first + i
        n, H, D = q.shape
        L, Hkv, _ = keys.shape
        o = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
        hidden = torch.arange(L, device="cuda")[None, :] > first + torch.arange(n, device="cuda")[:, None]
        for h in range(H):
            kv = h * Hkv // H
            logits = torch.einsum("id,jd->ij", q[:, h].double(), keys[:, kv]) / math.sqrt(D)
            p = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
            o[:, h] = torch.einsum("ij,jd->id", p, values[:, kv])
        return o

    def fp32(x):
        # the int8 format's scales, their ratios and quotients are fp32 numbers by definition: which
        # integer a value next to a border becomes follows from them
        return x.float().double()

    def appended(x):
        rows, pool = s[x].double(), s[x + "_pool"].double()
        scale = s[x + "_scale"].double() if c["kv"] == "i8" else None
        table = s["block_table"].tolist()
        for b in range(c["batch"]):
            at, t = total[b] - (cu[b + 1] - cu[b]), cu[b]
            while at < total[b]:
                block, r0 = table[b][at // page], at % page
                n = min(page - r0, total[b] - at)
                new = rows[t:t + n].transpose(0, 1)
                if scale is None:
                    pool[block, :, r0:r0 + n] = new
                else:
                    per = fp32(new.abs().amax((1, 2)) / 127)
                    if r0:
                        before = scale[block].clone()
                        per = torch.maximum(per, before)
                        kept = pool[block, :, :r0] * fp32(before / per)[:, None, None]
                        pool[block, :, :r0] = torch.round(fp32(kept))
                    scale[block] = per
                    pool[block, :, r0:r0 + n] = torch.round(fp32(new / per[:, None, None]))
                at, t = at + n, t + n
        return (pool, None) if scale is None else (pool * scale[:, :, None, None], scale)

    if c["op"] == "plan":
        return None
    s = prepare(c, seed)
    cu, total, page = s["cu_new"].tolist(), s["total_lens"].tolist(), c["page"]
    if c["op"] == "append":
        (k, ks), (v, vs) = appended("k"), appended("v")
        return (k, v) if ks is None else (k, v, ks, vs)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        t0, t1 = cu[b], cu[b + 1]
        if c["op"] == "prompt":
            keys, values, first = s["k"][t0:t1].double(), s["v"][t0:t1].double(), 0
        else:
            first, got = total[b] - (t1 - t0), []
            ids = s["block_table"][b, :_up(total[b], page)].long()
            for x in "kv":
                y = s[x + "_pool"][ids].double()
                if c["kv"] == "i8":
                    y = y * s[x + "_scale"][ids].double()[:, :, None, None]
                got.append(y.permute(0, 2, 1, 3).reshape(-1, c["kv_heads"], c["dim"])[:total[b]])
            keys, values = got
        out[t0:t1] = attention(s["q"][t0:t1], keys, values, first)
    return out
