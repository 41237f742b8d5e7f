"""Torch-facing convenience over the stream-level C ABI.

``PagedDecoder`` launches ``kvb_paged_decode_async`` on torch's current CUDA stream with torch
tensors as device buffers; torch is only the allocator and stream here, the work is the library's
CUDA kernels. ``plan_step``, ``append_kv``, ``append_kv_i8`` and ``PagedPrefill`` are the steps around
it, for several new tokens per sequence: they run on the device that holds their tensors, on its
current stream, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import torch

from . import Kernel, KvType, Shape, _CAppendArgs, _CChunkArgs, _CPromptArgs, _CShape, _CStepPlanArgs, device_args, \
    paged_append, paged_chunk_async, paged_chunk_workspace_bytes, paged_decode_async, paged_error_flag, \
    paged_part_tokens, paged_workspace_bytes, prompt_async, prompt_workspace_bytes, step_plan


_KV_DTYPE = {KvType.f32: torch.float32, KvType.f16: torch.float16, KvType.i8: torch.int8}


def kv_type_of(t: torch.Tensor) -> KvType:
    for k, v in _KV_DTYPE.items():
        if t.dtype == v:
            return k
    raise ValueError(f"unsupported cache dtype {t.dtype}")


class PagedDecoder:
    """One decode step per call over a paged cache held in torch tensors.

    q: float32 [B][H][D]; k_pool, v_pool: [num_blocks][Hkv][page][D] (float32, float16 or int8);
    block_table: int32 [B][max_blocks]; seq_lens: int32 [B]; k_scale, v_scale: float32
    [num_blocks][Hkv] for int8. The workspace is owned by the decoder (grown and zeroed on demand);
    calls on one decoder must not overlap on the device.
    """

    def __init__(self, device: Optional[torch.device] = None):
        self.device = torch.device(device or torch.device("cuda", torch.cuda.current_device()))
        self.workspace = torch.zeros(256, dtype=torch.uint8, device=self.device)

    def args(self, q, k_pool, v_pool, block_table, seq_lens, max_len, *, out, k_scale=None, v_scale=None,
             part_tokens=0, share_kv=True, kernel=Kernel.auto, tables_ready=False, inputs_ready=False,
             step_stream=False):
        B, H, D = q.shape
        num_blocks, Hkv, page, D2 = k_pool.shape
        if D2 != D or v_pool.shape != k_pool.shape:
            raise ValueError("pool shapes do not match q")
        for t in (q, k_pool, v_pool, block_table, seq_lens, out):
            if not t.is_contiguous() or t.device != self.device:
                raise ValueError("tensors must be contiguous and on the decoder's device")
        kvt = kv_type_of(k_pool)
        return device_args(Shape(B, H, Hkv, D), kvt, page, block_table.shape[1], int(max_len), q=q.data_ptr(),
                           k=k_pool.data_ptr(), v=v_pool.data_ptr(), block_table=block_table.data_ptr(),
                           seq_lens=seq_lens.data_ptr(), out=out.data_ptr(), num_blocks=num_blocks,
                           part_tokens=part_tokens, share_kv=share_kv,
                           k_scale=k_scale.data_ptr() if k_scale is not None else 0,
                           v_scale=v_scale.data_ptr() if v_scale is not None else 0, kernel=kernel,
                           tables_ready=tables_ready, inputs_ready=inputs_ready, step_stream=step_stream)

    def __call__(self, q, k_pool, v_pool, block_table, seq_lens, max_len, *, k_scale=None, v_scale=None,
                 part_tokens=0, share_kv=True, kernel=Kernel.auto, out=None, stream=None, tables_ready=False,
                 inputs_ready=False, step_stream=False):
        if out is None:
            out = torch.empty_like(q)
        c = self.args(q, k_pool, v_pool, block_table, seq_lens, max_len, out=out, k_scale=k_scale,
                      v_scale=v_scale, part_tokens=part_tokens, share_kv=share_kv, kernel=kernel,
                      tables_ready=tables_ready, inputs_ready=inputs_ready, step_stream=step_stream)
        need = paged_workspace_bytes(c)
        if need > self.workspace.numel():
            self.workspace = torch.zeros(need, dtype=torch.uint8, device=self.device)
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        paged_decode_async(c, self.workspace.data_ptr(), self.workspace.numel(), s.cuda_stream)
        return out

    def part_tokens(self, q, k_pool, v_pool, block_table, seq_lens, max_len, **kw) -> int:
        out = torch.empty_like(q)
        return paged_part_tokens(self.args(q, k_pool, v_pool, block_table, seq_lens, max_len, out=out, **kw))

    def error_flag(self, stream=None) -> int:
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        return paged_error_flag(self.workspace.data_ptr(), s.cuda_stream)


# ---- serving steps of several new tokens per sequence ------------------------------------------------
# These calls sit on a decode step's critical path, a few microseconds of GPU work each: the checks below
# are written for little host time.

_NO_GUARD = contextlib.nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream
_INT32, _INT64, _F32, _I8 = torch.int32, torch.int64, torch.float32, torch.int8
_KV_TYPE = {v: int(k) for k, v in _KV_DTYPE.items()}


def _on(index: int):
    """Makes device `index` current for a launch (nothing to do where it is already)."""
    return _NO_GUARD if index == torch.cuda.current_device() else torch.cuda.device(index)


def _type(name: str, t) -> int:
    k = _KV_TYPE.get(t.dtype)
    if k is None:
        raise ValueError(f"unsupported {name} dtype {t.dtype}")
    return k


def _bound(n) -> int:
    """A bound on lengths as the C int it is passed in: any larger one says as much as the largest."""
    return max(-1, min(int(n), 0x7fffffff))


def _tensor(name: str, t, dtype, index: int, shape) -> int:
    """The address of a contiguous tensor of this type, device and shape."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index}")
    return t.data_ptr()


def _rows(name: str, t, index: int) -> int:
    """The token stride of [tokens][heads][dim] rows; a token's own values lie together."""
    if t.dim() == 3 and t.get_device() == index:
        a, b, c = t.stride()
        if c == 1 and (b == t.shape[2] or t.shape[1] == 1):
            return a
    raise ValueError(f"{name} must be [tokens][heads][dim] on cuda:{index}, with each token's heads contiguous")


def _error(error_word, index: int):
    if error_word is None:
        return None
    if error_word.dtype not in (torch.int32, torch.uint32) or error_word.get_device() != index or error_word.numel() < 1:
        raise ValueError(f"error_word must be an int32 tensor on cuda:{index}")
    return error_word.data_ptr()


def _table(block_table, batch: int, index: int):
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be [batch][max_blocks]")
    return _tensor("block_table", block_table, _INT32, index, block_table.shape), block_table.shape[1]


class StepPlan(NamedTuple):
    """What ``plan_step`` returns (include/kvb_cuda.h, kvb_step_plan_args)."""
    total_lens: torch.Tensor  # int32 [batch], -1: refused
    cu_new: torch.Tensor      # int32 [batch + 1]
    slot_map: torch.Tensor    # int64 [num_tokens], -1: no slot
    positions: torch.Tensor   # int32 [num_tokens]
    ring_pos: torch.Tensor    # int64 [2]: head after the step, tail


def plan_step(seq_lens, new_lens, block_table, ring, ring_pos, *, page_size: int, num_blocks: int, num_tokens: int,
              error_word=None) -> StepPlan:
    """Pages and slots of a step's new tokens (kvb_step_plan), from the tokens cached (`seq_lens`) and
    added (`new_lens`) per sequence, both int32 [batch].

    Free block ids are ``ring[head % n], ..`` up to ``tail`` with ``ring_pos = [head, tail]`` (int64); new
    ids are written into `block_table` (int32 [batch][max_blocks]). The next step's `ring_pos` is the
    plan's; ids of finished requests go back with ``ring[(tail + torch.arange(m)) % n] = ids`` and
    ``ring_pos[1] += m``. `num_tokens` is the length of the packed step (the sum of `new_lens`, or more).
    `error_word`, an int32 tensor, collects the error bits.
    """
    index = seq_lens.get_device()
    if index < 0:
        raise ValueError("plan_step takes CUDA tensors")
    page_size, num_blocks, num_tokens = int(page_size), int(num_blocks), int(num_tokens)
    if not 0 <= num_tokens < 1 << 31 or seq_lens.dim() != 1 or ring.dim() != 1:
        raise ValueError("num_tokens outside [0, 2^31), or seq_lens or ring not one-dimensional")
    if not 0 < page_size < 1 << 31:
        raise ValueError("page_size must be in [1, 2^31)")
    batch = seq_lens.shape[0]
    lens = _tensor("seq_lens", seq_lens, _INT32, index, (batch,))
    pos = _tensor("ring_pos", ring_pos, _INT64, index, (2,))
    table, max_blocks = _table(block_table, batch, index)
    p = StepPlan(torch.empty_like(seq_lens), seq_lens.new_empty(batch + 1), ring_pos.new_empty(num_tokens),
                 seq_lens.new_empty(num_tokens), torch.empty_like(ring_pos))
    a = _CStepPlanArgs(batch, page_size, max_blocks, num_tokens, lens,
                       _tensor("new_lens", new_lens, _INT32, index, (batch,)), table,
                       _tensor("ring", ring, _INT32, index, ring.shape), pos, p.ring_pos.data_ptr(),
                       p.total_lens.data_ptr(), p.cu_new.data_ptr(), p.slot_map.data_ptr(), p.positions.data_ptr(),
                       ring.shape[0], num_blocks, _error(error_word, index))
    with _on(index):
        step_plan(a, _raw_stream(index))
    return p


def _append(k, v, k_pool, v_pool, index, slots, batch, max_blocks, scales, lists, error_word):
    if k.shape != v.shape or k.dtype is not v.dtype:
        raise ValueError("k and v must have one shape and type")
    k_stride, v_stride = _rows("k", k, index), _rows("v", v, index)
    T, Hkv, D = k.shape
    pool = k_pool.shape
    if len(pool) != 4 or pool[1] != Hkv or pool[3] != D:
        raise ValueError("pools must be [num_blocks][kv_heads][page][dim], heads and dim those of k")
    a = _CAppendArgs(_CShape(batch, Hkv, Hkv, D), _type("k", k), _type("pool", k_pool), pool[2], max_blocks, T,
                     k.data_ptr(), v.data_ptr(), k_stride, v_stride,
                     _tensor("k_pool", k_pool, k_pool.dtype, index, pool),
                     _tensor("v_pool", v_pool, k_pool.dtype, index, pool), *scales, pool[0], slots, *lists,
                     _error(error_word, index))
    with _on(index):
        paged_append(a, _raw_stream(index))


def append_kv(k, v, k_pool, v_pool, *, slot_map, error_word=None) -> None:
    """New tokens' keys and values (fp32 or fp16 [tokens][kv_heads][dim], any token stride of whole 16
    bytes) into fp32 or fp16 pages, at the plan's `slot_map` (kvb_paged_append)."""
    if k_pool.dtype is _I8:
        raise ValueError("int8 pages are written by append_kv_i8")
    index = k_pool.get_device()
    if index < 0:
        raise ValueError("the pools must be CUDA tensors")
    slots = _tensor("slot_map", slot_map, _INT64, index, k.shape[:1])
    _append(k, v, k_pool, v_pool, index, slots, 0, 0, (None, None), (None, None, None), error_word)


def append_kv_i8(k, v, k_pool, v_pool, k_scale, v_scale, *, block_table, total_lens, cu_new, error_word=None) -> None:
    """New tokens' keys and values quantized into int8 pages; the scales ([num_blocks][kv_heads]) and
    the rows of pages that were begun follow where a larger value needs it (kvb_paged_append)."""
    if k_pool.dtype is not _I8:
        raise ValueError("append_kv_i8 writes int8 pages")
    index, batch = k_pool.get_device(), total_lens.shape[0]
    if index < 0:
        raise ValueError("the pools must be CUDA tensors")
    table, max_blocks = _table(block_table, batch, index)
    if batch == 0:
        if k.shape[0]:
            raise ValueError("tokens without a sequence")
        return
    scales = k_pool.shape[:2]
    _append(k, v, k_pool, v_pool, index, None, batch, max_blocks,
            (_tensor("k_scale", k_scale, _F32, index, scales), _tensor("v_scale", v_scale, _F32, index, scales)),
            (table, _tensor("total_lens", total_lens, _INT32, index, (batch,)),
             _tensor("cu_new", cu_new, _INT32, index, (batch + 1,))), error_word)


class PagedPrefill:
    """Attention of several new tokens per sequence: ``chunk`` over the paged cache, ``prompt`` over whole
    packed prompts. q (and out) fp32 or fp16 [tokens][heads][dim]. Each call takes its workspace from
    torch's allocator on the stream it runs on, so calls may overlap on different streams; the object
    keeps only the error word that they share.
    """

    def __init__(self, device: Optional[torch.device] = None):
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.error_word = torch.zeros(1, dtype=torch.int32, device=self.device)

    def _run(self, a, workspace_bytes, launch, index):
        with _on(index):
            n = workspace_bytes(a)
            workspace = self.error_word.new_empty((n + 3) // 4)
            launch(a, workspace.data_ptr(), n, _raw_stream(index))

    def chunk(self, q, k_pool, v_pool, block_table, total_lens, cu_new, *, max_new: int, max_len: int, k_scale=None,
              v_scale=None, out=None, kernel=Kernel.auto):
        """New token i of sequence b (packed row cu_new[b] + i) over the tokens at positions up to its own,
        total_lens[b] - n_b + i; the pages hold the new tokens already (kvb_paged_chunk_async)."""
        index = self.device.index
        q_stride = _rows("q", q, index)
        T, H, D = q.shape
        pool = k_pool.shape
        if len(pool) != 4 or pool[3] != D:
            raise ValueError("pools must be [num_blocks][kv_heads][page][dim], dim that of q")
        batch = total_lens.shape[0]
        table, max_blocks = _table(block_table, batch, index)
        if out is None:
            out = q.new_empty(q.shape)
        ks = None if k_scale is None else _tensor("k_scale", k_scale, _F32, index, pool[:2])
        vs = None if v_scale is None else _tensor("v_scale", v_scale, _F32, index, pool[:2])
        a = _CChunkArgs(_CShape(batch, H, pool[1], D), _type("q", q), _type("pool", k_pool), pool[2], max_blocks, T,
                        _bound(max_new), _bound(max_len), q.data_ptr(), q_stride,
                        _tensor("k_pool", k_pool, k_pool.dtype, index, pool),
                        _tensor("v_pool", v_pool, k_pool.dtype, index, pool), ks, vs, pool[0], table,
                        _tensor("total_lens", total_lens, _INT32, index, (batch,)),
                        _tensor("cu_new", cu_new, _INT32, index, (batch + 1,)),
                        _tensor("out", out, q.dtype, index, q.shape), self.error_word.data_ptr(), kernel)
        self._run(a, paged_chunk_workspace_bytes, paged_chunk_async, index)
        return out

    def prompt(self, q, k, v, cu_lens, *, max_len: int, out=None, kernel=Kernel.auto):
        """Causal attention of packed prompts, prompt b being rows cu_lens[b] .. cu_lens[b + 1) of q, k
        and v (one type; token strides may differ), at most max_len tokens each (kvb_prompt_async)."""
        index = self.device.index
        if k.shape != v.shape or k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[-1]:
            raise ValueError("k and v must have one shape, with q's tokens and dim")
        if k.dtype is not q.dtype or v.dtype is not q.dtype:
            raise ValueError("q, k and v must have one type")
        q_stride, k_stride, v_stride = _rows("q", q, index), _rows("k", k, index), _rows("v", v, index)
        T, H, D = q.shape
        if out is None:
            out = q.new_empty(q.shape)
        a = _CPromptArgs(_CShape(cu_lens.shape[0] - 1, H, k.shape[1], D), _type("q", q), T, _bound(max_len), q.data_ptr(),
                         k.data_ptr(), v.data_ptr(), q_stride, k_stride, v_stride,
                         _tensor("cu_lens", cu_lens, _INT32, index, (cu_lens.shape[0],)),
                         _tensor("out", out, q.dtype, index, q.shape), self.error_word.data_ptr(), kernel)
        self._run(a, prompt_workspace_bytes, prompt_async, index)
        return out

    def error_flag(self) -> int:
        """Reads and clears the error bits of the calls so far (waits for the current stream): 1 bad
        length, 2 bad block id, 4 a device wait gave up."""
        flag = int(self.error_word.item())
        if flag:
            self.error_word.zero_()
        return flag
