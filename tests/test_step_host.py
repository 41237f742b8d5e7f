"""CPU checks of the serving-step entry points (plan, append, chunk and prompt attention): struct
layouts against the header, and refusals with KVB_ERR_INVALID before any device is touched."""
import ctypes

import pytest

import kv_cache_bench_b200 as kvb
from tests.test_capi import _c_layout

K = kvb.KvType


@pytest.mark.parametrize("struct,cls", [("kvb_step_plan_args", "_CStepPlanArgs"), ("kvb_append_args", "_CAppendArgs"),
                                        ("kvb_chunk_args", "_CChunkArgs"), ("kvb_prompt_args", "_CPromptArgs")])
def test_python_structs_match_the_header_layout(struct, cls):
    c = getattr(kvb, cls)
    names = [f[0] for f in c._fields_]
    got = _c_layout(struct, names)
    assert got == [ctypes.sizeof(c)] + [getattr(c, n).offset for n in names], struct


def plan_args(batch=2, page=16, max_blocks=4, tokens=8, **over):
    kw = dict(seq_lens=0x1000, new_lens=0x2000, block_table=0x3000, ring=0x4000, ring_pos=0x5000, ring_out=0x6000,
              total_lens=0x7000, cu_new=0x8000, slot_map=0x9000, positions=0xa000, ring_size=8, num_blocks=8)
    kw.update(over)
    return kvb.step_plan_args(batch, page, max_blocks, tokens, **kw)


@pytest.mark.parametrize("a,msg", [
    (plan_args(page=0), "page_size"), (plan_args(batch=-1), "batch"), (plan_args(tokens=-1), "num_tokens"),
    (plan_args(max_blocks=-1), "max_blocks"), (plan_args(num_blocks=0), "num_blocks"),
    (plan_args(ring_size=-1), "ring_size"), (plan_args(ring=0), "null"), (plan_args(ring_pos=0), "null"),
    (plan_args(seq_lens=0), "null"), (plan_args(total_lens=0), "null"), (plan_args(cu_new=0), "null"),
    (plan_args(block_table=0), "null"), (plan_args(slot_map=0), "null"),
    (plan_args(total_lens=0x1000), "an output overlaps an input"),  # seq_lens in place
    (plan_args(ring_out=0x5008), "an output overlaps an input"),    # half of ring_pos in place
    (plan_args(block_table=0x4010), "an output overlaps an input"),
    (plan_args(slot_map=0x9fc8), "two outputs overlap"),            # its last entry is positions' first
])
def test_plan_refusals(a, msg):
    with pytest.raises(ValueError, match=msg):
        kvb.step_plan(a)


def append_args(batch=2, hkv=2, dim=128, src=K.f16, kv=K.f16, page=16, tokens=4, **over):
    kw = dict(k=0x1000, v=0x2000, k_stride=hkv * dim, v_stride=hkv * dim, k_pool=0x3000, v_pool=0x4000, num_blocks=4,
              slot_map=0x5000, k_scale=0x6000, v_scale=0x7000, max_blocks=4, block_table=0x8000, total_lens=0x9000,
              cu_new=0xa000)
    kw.update(over)
    return kvb.append_args(batch, hkv, dim, src, kv, page, tokens, **kw)


@pytest.mark.parametrize("a,msg", [
    (append_args(src=K.i8), "rows must be"), (append_args(kv=K.f32), "takes f32 rows"), (append_args(dim=100), "head_dim"),
    (append_args(dim=0, k_stride=8, v_stride=8), "head_dim"), (append_args(hkv=0), "num_kv_heads"),
    (append_args(page=0), "page_size"), (append_args(tokens=-1), "num_tokens"), (append_args(num_blocks=0), "num_blocks"),
    (append_args(k=0), "null"), (append_args(v_pool=0), "null"), (append_args(k=0x1008), "16-byte"),
    (append_args(k_pool=0x3004), "16-byte"), (append_args(k_stride=255), "stride"), (append_args(v_stride=260), "stride"),
    (append_args(slot_map=0), "slot_map"), (append_args(kv=K.i8, k_scale=0), "scales"),
    (append_args(kv=K.i8, cu_new=0), "cu_new"), (append_args(kv=K.i8, batch=0), "batch"), (append_args(batch=-1), "batch"),
    (append_args(page=1 << 24), "2\\^31"),
])
def test_append_refusals(a, msg):
    with pytest.raises(ValueError, match=msg):
        kvb.paged_append(a)


def test_append_of_no_tokens_is_nothing():
    kvb.paged_append(append_args(tokens=0, k=0, v=0, slot_map=0))


def chunk_args(shape=kvb.Shape(2, 8, 2, 128), q=K.f16, kv=K.f16, page=16, max_blocks=4, tokens=6, max_new=4, max_len=64,
               kernel=kvb.Kernel.auto, **over):
    kw = dict(q=0x1000, q_stride=1024, k=0x2000, v=0x3000, num_blocks=8, block_table=0x4000, total_lens=0x5000,
              cu_new=0x6000, out=0x7000, error_word=0x8000, k_scale=0x9000, v_scale=0xa000)
    kw["q"] = over.pop("qp", kw["q"])
    kw.update(over)
    return kvb.chunk_args(shape, q, kv, page, max_blocks, tokens, max_new, max_len, kernel=kernel, **kw)


@pytest.mark.parametrize("a,msg", [
    (chunk_args(shape=kvb.Shape(2, 8, 2, 96)), "head_dim"), (chunk_args(shape=kvb.Shape(2, 6, 4, 128)), "Hkv"),
    (chunk_args(shape=kvb.Shape(-1, 8, 2, 128)), "shape"), (chunk_args(shape=kvb.Shape(1, 130, 2, 128)), "64 query heads"),
    (chunk_args(q=K.i8), "f32 or f16"), (chunk_args(page=0), "page_size"), (chunk_args(max_new=0), "max_new"),
    (chunk_args(max_len=-1), "max_len"), (chunk_args(tokens=-1), "num_tokens"), (chunk_args(num_blocks=0), "num_blocks"),
    (chunk_args(kv=K.i8, v_scale=0), "scales"), (chunk_args(error_word=0), "null"), (chunk_args(out=0), "null"),
    (chunk_args(qp=0), "null"), (chunk_args(qp=0x1008), "16-byte"), (chunk_args(q_stride=1000), "stride"),
    (chunk_args(q_stride=1028), "stride"), (chunk_args(out=0x7004), "32-byte"), (chunk_args(out=0x7010), "32-byte"), (chunk_args(k=0x2008), "16-byte"),
    (chunk_args(kernel=kvb.Kernel.mma), "kernel"),
])
def test_chunk_refusals(a, msg):
    with pytest.raises(ValueError, match=msg):
        kvb.paged_chunk_async(a, 0x10000, 1 << 30)
    with pytest.raises(ValueError, match=msg):
        kvb.paged_chunk_workspace_bytes(a)


def prompt_args(shape=kvb.Shape(2, 8, 2, 64), type=K.f16, tokens=6, max_len=4, kernel=kvb.Kernel.auto, **over):
    kw = dict(q=0x1000, k=0x2000, v=0x3000, q_stride=768, k_stride=768, v_stride=768, cu_lens=0x4000, out=0x5000,
              error_word=0x6000)
    kw.update(over)
    return kvb.prompt_args(shape, type, tokens, max_len, kernel=kernel, **kw)


@pytest.mark.parametrize("a,msg", [
    (prompt_args(type=K.i8), "f32 or f16"), (prompt_args(max_len=0), "max_new"), (prompt_args(q_stride=511), "stride"),
    (prompt_args(k_stride=127), "stride"), (prompt_args(v_stride=132), "stride"), (prompt_args(k=0x2004), "16-byte"),
    (prompt_args(out=0x5010), "32-byte"), (prompt_args(cu_lens=0), "null"), (prompt_args(v=0), "null"), (prompt_args(shape=kvb.Shape(2, 8, 2, 80)), "head_dim"),
])
def test_prompt_refusals(a, msg):
    with pytest.raises(ValueError, match=msg):
        kvb.prompt_async(a, 0x10000, 1 << 30)


def test_calls_without_tokens_need_no_device():
    kvb.paged_chunk_async(chunk_args(tokens=0, qp=0, out=0), 0, 0)
    kvb.paged_chunk_async(chunk_args(shape=kvb.Shape(0, 8, 2, 128)), 0, 0)
    kvb.prompt_async(prompt_args(tokens=0, max_len=0, q=0, k=0, v=0, out=0), 0, 0)
    assert kvb.paged_chunk_workspace_bytes(chunk_args(tokens=0)) <= 4096
