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

from . import Kernel, KvType, Shape, append_args, chunk_args, device_args, paged_append, paged_chunk_async, \
    paged_chunk_workspace_bytes, paged_decode_async, paged_error_flag, paged_part_tokens, paged_workspace_bytes, \
    prompt_args, prompt_async, prompt_workspace_bytes, step_plan, step_plan_args

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

_NO_GUARD = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes `device` current for a launch (nothing to do where it is already)."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _tensor(name: str, t, dtype, device, shape=None) -> int:
    """The address of a contiguous tensor of this type, place and shape."""
    if t.dtype is not dtype or t.device != device or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor"
                         f"{'' if shape is None else ' of shape ' + str(tuple(shape))} on {device}")
    return t.data_ptr()


def _rows(name: str, t, device) -> int:
    """The token stride of [tokens][heads][dim] rows; a token's own values lie together."""
    if t.dim() != 3 or t.device != device or t.stride(2) != 1 or t.stride(1) != t.shape[2]:
        raise ValueError(f"{name} must be [tokens][heads][dim] on {device}, with each token's heads contiguous")
    return t.stride(0)


def _error(error_word, device) -> int:
    if error_word is None:
        return 0
    if error_word.dtype not in (torch.int32, torch.uint32) or error_word.device != device or error_word.numel() < 1:
        raise ValueError(f"error_word must be an int32 tensor on {device}")
    return error_word.data_ptr()


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
    device = seq_lens.device
    if device.type != "cuda":
        raise ValueError("plan_step takes CUDA tensors")
    batch = seq_lens.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be [batch][max_blocks]")
    if num_tokens < 0:
        raise ValueError("num_tokens < 0")
    new = lambda n, dtype: torch.empty(n, dtype=dtype, device=device)  # noqa: E731
    p = StepPlan(new(batch, torch.int32), new(batch + 1, torch.int32), new(num_tokens, torch.int64),
                 new(num_tokens, torch.int32), new(2, torch.int64))
    a = step_plan_args(
        batch, page_size, block_table.shape[1], num_tokens,
        seq_lens=_tensor("seq_lens", seq_lens, torch.int32, device, (batch,)),
        new_lens=_tensor("new_lens", new_lens, torch.int32, device, (batch,)),
        block_table=_tensor("block_table", block_table, torch.int32, device),
        ring=_tensor("ring", ring, torch.int32, device), ring_pos=_tensor("ring_pos", ring_pos, torch.int64, device, (2,)),
        ring_out=p.ring_pos.data_ptr(), total_lens=p.total_lens.data_ptr(), cu_new=p.cu_new.data_ptr(),
        slot_map=p.slot_map.data_ptr(), positions=p.positions.data_ptr(), ring_size=ring.numel(),
        num_blocks=num_blocks, error_word=_error(error_word, device))
    with _on(device):
        step_plan(a, _stream(device))
    return p


def _append(k, v, k_pool, v_pool, error_word, batch=0, **kw):
    device = k_pool.device
    if device.type != "cuda":
        raise ValueError("the pools must be CUDA tensors")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must have one shape and type")
    k_stride, v_stride = _rows("k", k, device), _rows("v", v, device)
    if k_pool.dim() != 4 or k_pool.shape[1] != k.shape[1] or k_pool.shape[3] != k.shape[2]:
        raise ValueError("pools must be [num_blocks][kv_heads][page][dim], heads and dim those of k")
    _tensor("v_pool", v_pool, k_pool.dtype, device, k_pool.shape)
    _tensor("k_pool", k_pool, k_pool.dtype, device)
    a = append_args(batch, k.shape[1], k.shape[2], kv_type_of(k), kv_type_of(k_pool), k_pool.shape[2], k.shape[0],
                    k=k.data_ptr(), v=v.data_ptr(), k_stride=k_stride, v_stride=v_stride, k_pool=k_pool.data_ptr(),
                    v_pool=v_pool.data_ptr(), num_blocks=k_pool.shape[0], error_word=_error(error_word, device), **kw)
    with _on(device):
        paged_append(a, _stream(device))


def append_kv(k, v, k_pool, v_pool, *, slot_map, error_word=None) -> None:
    """New tokens' keys and values (fp32 or fp16 [tokens][kv_heads][dim], any token stride of whole 16
    bytes) into fp32 or fp16 pages, at the plan's `slot_map` (kvb_paged_append)."""
    if k_pool.dtype == torch.int8:
        raise ValueError("int8 pages are written by append_kv_i8")
    _append(k, v, k_pool, v_pool, error_word,
            slot_map=_tensor("slot_map", slot_map, torch.int64, k_pool.device, (k.shape[0],)))


def append_kv_i8(k, v, k_pool, v_pool, k_scale, v_scale, *, block_table, total_lens, cu_new, error_word=None) -> None:
    """New tokens' keys and values quantized into int8 pages; the scales ([num_blocks][kv_heads]) and
    the rows of pages that were begun follow where a larger value needs it (kvb_paged_append)."""
    if k_pool.dtype != torch.int8:
        raise ValueError("append_kv_i8 writes int8 pages")
    device, batch = k_pool.device, total_lens.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError("block_table must be [batch][max_blocks]")
    if batch == 0:
        if k.shape[0]:
            raise ValueError("tokens without a sequence")
        return
    scale = lambda n, t: _tensor(n, t, torch.float32, device, k_pool.shape[:2])  # noqa: E731
    _append(k, v, k_pool, v_pool, error_word, batch, k_scale=scale("k_scale", k_scale),
            v_scale=scale("v_scale", v_scale), max_blocks=block_table.shape[1],
            block_table=_tensor("block_table", block_table, torch.int32, device),
            total_lens=_tensor("total_lens", total_lens, torch.int32, device, (batch,)),
            cu_new=_tensor("cu_new", cu_new, torch.int32, device, (batch + 1,)))


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

    def _out(self, q, out):
        if out is None:
            return torch.empty(q.shape, dtype=q.dtype, device=self.device)
        _tensor("out", out, q.dtype, self.device, q.shape)
        return out

    def chunk(self, q, k_pool, v_pool, block_table, total_lens, cu_new, *, max_new: int, max_len: int, k_scale=None,
              v_scale=None, out=None, kernel=Kernel.auto):
        """New token i of sequence b (packed row cu_new[b] + i) over the tokens at positions up to its own,
        total_lens[b] - n_b + i; the pages hold the new tokens already (kvb_paged_chunk_async)."""
        device = self.device
        q_stride = _rows("q", q, device)
        T, H, D = q.shape
        if k_pool.dim() != 4 or k_pool.shape[3] != D:
            raise ValueError("pools must be [num_blocks][kv_heads][page][dim], dim that of q")
        num_blocks, Hkv, page, _ = k_pool.shape
        batch = total_lens.shape[0]
        if block_table.dim() != 2 or block_table.shape[0] != batch:
            raise ValueError("block_table must be [batch][max_blocks]")
        out = self._out(q, out)
        scale = lambda n, t: 0 if t is None else _tensor(n, t, torch.float32, device, (num_blocks, Hkv))  # noqa: E731
        a = chunk_args(Shape(batch, H, Hkv, D), kv_type_of(q), kv_type_of(k_pool), page, block_table.shape[1], T,
                       int(max_new), int(max_len), q=q.data_ptr(), q_stride=q_stride,
                       k=_tensor("k_pool", k_pool, k_pool.dtype, device),
                       v=_tensor("v_pool", v_pool, k_pool.dtype, device, k_pool.shape), num_blocks=num_blocks,
                       block_table=_tensor("block_table", block_table, torch.int32, device),
                       total_lens=_tensor("total_lens", total_lens, torch.int32, device, (batch,)),
                       cu_new=_tensor("cu_new", cu_new, torch.int32, device, (batch + 1,)), out=out.data_ptr(),
                       error_word=self.error_word.data_ptr(), k_scale=scale("k_scale", k_scale),
                       v_scale=scale("v_scale", v_scale), kernel=kernel)
        with _on(device):
            n = paged_chunk_workspace_bytes(a)
            workspace = torch.empty(n, dtype=torch.uint8, device=device)
            paged_chunk_async(a, workspace.data_ptr(), n, _stream(device))
        return out

    def prompt(self, q, k, v, cu_lens, *, max_len: int, out=None, kernel=Kernel.auto):
        """Causal attention of packed prompts, prompt b being rows cu_lens[b] .. cu_lens[b + 1) of q, k
        and v (one type; token strides may differ), at most max_len tokens each (kvb_prompt_async)."""
        device = self.device
        if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
            raise ValueError("k and v must have one shape, with q's tokens and dim")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError("q, k and v must have one type")
        q_stride, k_stride, v_stride = _rows("q", q, device), _rows("k", k, device), _rows("v", v, device)
        T, H, D = q.shape
        out = self._out(q, out)
        a = prompt_args(Shape(cu_lens.shape[0] - 1, H, k.shape[1], D), kv_type_of(q), T, int(max_len),
                        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=q_stride, k_stride=k_stride,
                        v_stride=v_stride, cu_lens=_tensor("cu_lens", cu_lens, torch.int32, device),
                        out=out.data_ptr(), error_word=self.error_word.data_ptr(), kernel=kernel)
        with _on(device):
            n = prompt_workspace_bytes(a)
            workspace = torch.empty(n, dtype=torch.uint8, device=device)
            prompt_async(a, workspace.data_ptr(), n, _stream(device))
        return out

    def error_flag(self) -> int:
        """Reads and clears the error bits of the calls so far (waits for the current stream): 1 bad
        length, 2 bad block id, 4 a device wait gave up."""
        flag = int(self.error_word.item())
        if flag:
            self.error_word.zero_()
        return flag
