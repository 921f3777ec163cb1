"""Paged K/V cache in 8 bits and the attention that reads it: the attention
side of the decoder layers whose MLPs the rest of the package runs.

    cache = KvCache(num_blocks, kv_heads, head_dim)              # one per layer
    batch = KvBatch(num_blocks, 16, max_requests=R, max_blocks=W, q_heads=Hq, kv_heads=H, head_dim=D)
    step = batch.plan(new_tokens, total, max_new=n)              # once per step, for every layer
    cache.append(k, v, step.slots)                               # per layer
    out = paged_attention(q, cache, step)                        # [total, Hq, D]
    batch.commit(finished)                                       # once per step

``KvBatch`` keeps the requests' lengths, block tables and free blocks on the
device; a step's plan is one kernel, and no call synchronises.  ``KvCache``
holds a layer's K and V codes with one scale per (block, head) for each; the
formats are described in ``nsmlp.h``.  The reference has no such cache: its
attention and K/V cache are torch code in ``streaming_llama_runtime.py``
(RT:5927-7142).  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._runtime import ptr, require_device, stream_handle, workspace

__all__ = ["KvCache", "KvBatch", "KvStep", "paged_attention"]

_FORMATS = {"int8": _lib.NSMLP_KV_INT8, "e4m3": _lib.NSMLP_KV_E4M3}
_DTYPES = {torch.float16: _lib.NSMLP_DTYPE_F16, torch.bfloat16: _lib.NSMLP_DTYPE_BF16}


def _device(device) -> torch.device:
    return require_device(torch.empty(0, device="cuda" if device is None else device), "cache")


def _rows(t: torch.Tensor, what: str, heads: int, dim: int, device: torch.device) -> torch.Tensor:
    """[tokens, heads, dim] in fp16 or bf16 that the kernels can read in 16-byte pieces; a copy where the strides do not allow it."""
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{what} must be fp16 or bf16, got {t.dtype}")
    if t.dim() != 3 or tuple(t.shape[1:]) != (heads, dim):
        raise RuntimeError(f"{what} must be [tokens, {heads}, {dim}], got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{what} must be on {device}, got {t.device}")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        t = t if t.data_ptr() % 16 == 0 else t.clone()
    return t


def _slots(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int64 or t.dim() != 1 or t.device != device:
        raise RuntimeError(f"slots must be an int64 [tokens] tensor on {device}")
    return t.contiguous()


class KvCache:
    """A layer's K and V: ``num_blocks`` blocks of ``block_tokens`` (16, 32 or
    64) tokens, ``fmt`` "int8" or "e4m3", ``head_dim`` 64 or 128."""

    def __init__(self, num_blocks: int, kv_heads: int, head_dim: int, *, block_tokens: int = 16, fmt: str = "int8",
                 device=None):
        if fmt not in _FORMATS:
            raise RuntimeError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
        if head_dim not in (64, 128):
            raise RuntimeError(f"head_dim must be 64 or 128, got {head_dim}")
        if block_tokens not in (16, 32, 64):
            raise RuntimeError(f"block_tokens must be 16, 32 or 64, got {block_tokens}")
        if num_blocks < 1 or kv_heads < 1:
            raise RuntimeError(f"num_blocks and kv_heads must be at least 1, got {num_blocks} and {kv_heads}")
        self.device = _device(device)
        self.num_blocks, self.kv_heads, self.head_dim = int(num_blocks), int(kv_heads), int(head_dim)
        self.block_tokens, self.fmt = int(block_tokens), fmt
        self.data = torch.zeros(num_blocks, kv_heads, 2, block_tokens * head_dim, dtype=torch.uint8, device=self.device)
        self.scale = torch.zeros(num_blocks, kv_heads, 2, dtype=torch.float32, device=self.device)
        self._view = _lib.KvCacheView(num_blocks=self.num_blocks, kv_heads=self.kv_heads, head_dim=self.head_dim,
                                      block_tokens=self.block_tokens, format=_FORMATS[fmt], data=ptr(self.data),
                                      scale=ptr(self.scale))

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store the rows ``k``, ``v`` [tokens, kv_heads, head_dim] at ``slots``
        (a plan's: a block's tokens stand next to each other, in order; a slot
        of -1 stores nothing).  Where the new rows exceed a block's scale its
        stored codes are rewritten under the larger one."""
        k = _rows(k, "k", self.kv_heads, self.head_dim, self.device)
        v = _rows(v, "v", self.kv_heads, self.head_dim, self.device)
        slots = _slots(slots, self.device)
        n = int(slots.numel())
        if k.dtype != v.dtype or int(k.shape[0]) != n or int(v.shape[0]) != n:
            raise RuntimeError(f"k, v and slots must be of the same length and k and v of one dtype: got {tuple(k.shape)} "
                               f"{k.dtype}, {tuple(v.shape)} {v.dtype} and {n} slots")
        _lib.call("nsmlp_kv_append", ctypes.byref(self._view), ptr(k), k.stride(0), k.stride(1), ptr(v), v.stride(0),
                  v.stride(1), _DTYPES[k.dtype], ptr(slots), n, stream_handle(self.device))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> dict[str, torch.Tensor]:
        """The stored rows at ``slots``: ``{"k": ..., "v": ...}`` of [tokens,
        kv_heads, head_dim] in ``dtype``; zeros for a slot of -1."""
        if dtype not in _DTYPES:
            raise RuntimeError(f"dtype must be fp16 or bf16, got {dtype}")
        slots = _slots(slots, self.device)
        n = int(slots.numel())
        out = torch.empty(2, n, self.kv_heads, self.head_dim, dtype=dtype, device=self.device)
        _lib.call("nsmlp_kv_read", ctypes.byref(self._view), ptr(slots), n, ptr(out[0]), ptr(out[1]), _DTYPES[dtype],
                  stream_handle(self.device))
        return {"k": out[0], "v": out[1]}


class KvStep:
    """A planned step: ``slots`` [total] int64 (-1: none), ``q_start``
    [requests + 1], ``kv_len`` [requests], ``info`` [4] = (ring head, free
    blocks, refused requests, sum of new tokens) after it, ``table`` the batch's
    block table.  ``info`` and the others are device tensors: reading them
    waits for the stream."""

    def __init__(self, batch: "KvBatch", total: int, max_new: int):
        R, dev = batch.requests, batch.device
        self.batch, self.total, self.max_new = batch, int(total), int(max_new)
        nbytes = int(_lib.lib().nsmlp_kv_schedule_bytes(ctypes.byref(batch._view), self.total, self.max_new))
        if nbytes == 0:
            raise RuntimeError(f"nsmlp_kv_schedule_bytes: {_lib.last_error()}")
        # one allocation: slots, then q_start, kv_len, next and info, then the schedule
        head = 8 * self.total
        ints = (3 * R + 5 + 3) // 4 * 4
        pad = -head % 16
        buf = torch.empty(head + pad + 4 * ints + nbytes, dtype=torch.uint8, device=dev)
        self.slots = buf[:head].view(torch.int64)
        v = buf[head + pad: head + pad + 4 * ints].view(torch.int32)
        self.q_start, self.kv_len, self._next, self.info = v[:R + 1], v[R + 1: 2 * R + 1], v[2 * R + 1: 3 * R + 1], \
            v[3 * R + 1: 3 * R + 5]
        base = ptr(buf) + head + pad
        self._buf = buf
        self._view = _lib.KvStepView(total=self.total, max_new=self.max_new, slots=ptr(buf), q_start=base,
                                     kv_len=base + 4 * (R + 1), next=base + 4 * (2 * R + 1), info=base + 4 * (3 * R + 1),
                                     schedule=base + 4 * ints, schedule_bytes=nbytes)
        self._ws_bytes: dict[int, int] = {}

    @property
    def table(self) -> torch.Tensor:
        return self.batch.table

    def workspace_bytes(self, head_dim: int) -> int:
        n = self._ws_bytes.get(head_dim)
        if n is None:
            n = int(_lib.lib().nsmlp_paged_attention_workspace_bytes(ctypes.byref(self.batch._view), self.total, self.max_new,
                                                                    head_dim))
            self._ws_bytes[head_dim] = n
        return n

    def check(self) -> None:
        """Wait for the plan and raise RuntimeError where it refused a request
        or its ``total`` is not the sum of the new tokens."""
        _, free, refused, total = self.info.tolist()
        if refused:
            raise RuntimeError(f"{refused} requests were refused: out of blocks ({free} are free), longer than the block table "
                               "or than max_new")
        if total != self.total:
            raise RuntimeError(f"the step was planned for {self.total} tokens, its requests bring {total}")


class KvBatch:
    """Lengths, block tables and free blocks of up to 4096 requests, on the
    device: ``cached`` [requests], ``table`` [requests, max_blocks] (-1: no
    block), and a ring of free block ids."""

    def __init__(self, num_blocks: int, block_tokens: int, *, max_requests: int, max_blocks: int, q_heads: int, kv_heads: int,
                 head_dim: int = 128, free_blocks: torch.Tensor | None = None, device=None):
        """``free_blocks``: the ids to hand out, in this order (default all, ascending)."""
        self.device = _device(device)
        self.requests, self.max_blocks, self.num_blocks = int(max_requests), int(max_blocks), int(num_blocks)
        self.block_tokens, self.q_heads, self.kv_heads, self.head_dim = int(block_tokens), int(q_heads), int(kv_heads), \
            int(head_dim)
        if self.requests < 1 or self.max_blocks < 1 or self.num_blocks < 1:
            raise RuntimeError("max_requests, max_blocks and num_blocks must be at least 1")
        self.cached = torch.zeros(self.requests, dtype=torch.int32, device=self.device)
        self.table = torch.full((self.requests, self.max_blocks), -1, dtype=torch.int32, device=self.device)
        ids = torch.arange(self.num_blocks, dtype=torch.int32, device=self.device)
        n_free = self.num_blocks
        if free_blocks is not None:
            n_free = int(free_blocks.numel())
            if n_free > self.num_blocks:
                raise RuntimeError(f"{n_free} free blocks of {self.num_blocks}")
            ids[:n_free] = free_blocks.to(device=self.device, dtype=torch.int32).reshape(-1)
        self.ring = ids
        self.state = torch.tensor([0, n_free], dtype=torch.int32, device=self.device)
        self._view = _lib.KvBatchView(requests=self.requests, max_blocks=self.max_blocks, num_blocks=self.num_blocks,
                                      block_tokens=self.block_tokens, q_heads=self.q_heads, kv_heads=self.kv_heads,
                                      cached=ptr(self.cached), table=ptr(self.table), ring=ptr(self.ring),
                                      state=ptr(self.state))
        if int(_lib.lib().nsmlp_kv_schedule_bytes(ctypes.byref(self._view), 1, 0)) == 0:
            raise RuntimeError(f"KvBatch: {_lib.last_error()}")
        self._step: KvStep | None = None

    def plan(self, new_tokens: torch.Tensor, total: int, *, max_new: int = 0, step: KvStep | None = None) -> KvStep:
        """Place the step's tokens: ``new_tokens`` [requests] int32 on the
        device (0 for a request that waits), ``total`` their sum, ``max_new``
        the most of one request where the caller knows it (it decides which
        kernels the attention launches).  Lengths and free blocks stay as they
        are until :meth:`commit`; a plan that is not committed can be made
        again.  ``step``: an earlier step of the same ``total`` and ``max_new``
        whose buffers are written again (a captured graph's)."""
        if new_tokens.dtype != torch.int32 or new_tokens.device != self.device or int(new_tokens.numel()) != self.requests \
                or not new_tokens.is_contiguous():
            raise RuntimeError(f"new_tokens must be a contiguous int32 [{self.requests}] tensor on {self.device}")
        if step is None:
            step = KvStep(self, total, max_new)
        elif step.batch is not self or step.total != int(total) or step.max_new != int(max_new):
            raise RuntimeError("the step to plan into belongs to another batch, total or max_new")
        _lib.call("nsmlp_kv_plan", ctypes.byref(self._view), ptr(new_tokens), ctypes.byref(step._view),
                  stream_handle(self.device))
        self._step = step
        return step

    def commit(self, finished: torch.Tensor | None = None) -> None:
        """Make the last plan's lengths the batch's, and end the requests with
        ``finished`` [requests] (int32, not 0): their blocks become free."""
        if finished is not None and (finished.dtype != torch.int32 or finished.device != self.device
                                     or int(finished.numel()) != self.requests or not finished.is_contiguous()):
            raise RuntimeError(f"finished must be a contiguous int32 [{self.requests}] tensor on {self.device}")
        st, self._step = self._step, None
        _lib.call("nsmlp_kv_commit", ctypes.byref(self._view), None if st is None else ctypes.byref(st._view), ptr(finished),
                  stream_handle(self.device))


def paged_attention(q: torch.Tensor, cache: KvCache, step: KvStep, *, scale: float | None = None,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    ws: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's queries ``q`` [total, q_heads, head_dim] (fp16 or
    bf16) over the cache, causal at the end of each request (its new tokens'
    K and V are appended before the call).  ``scale`` defaults to
    1/sqrt(head_dim).  Returns ``out`` [total, q_heads, head_dim]; ``lse``
    ([total, q_heads] fp32) receives the log of the softmax sums."""
    device = require_device(q, "q")
    b = step.batch
    if cache.device != device or b.device != device:
        raise RuntimeError(f"q is on {device}, the cache on {cache.device} and the batch on {b.device}")
    q = _rows(q, "q", b.q_heads, cache.head_dim, device)
    if int(q.shape[0]) != step.total:
        raise RuntimeError(f"q holds {int(q.shape[0])} tokens, the step {step.total}")
    shape = (step.total, b.q_heads, cache.head_dim)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=device)
    elif out.dtype != q.dtype or out.device != device or tuple(out.shape) != shape or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise RuntimeError(f"out must be a contiguous, 16-byte aligned {q.dtype} tensor {shape} on {device}")
    if lse is not None and (lse.dtype != torch.float32 or lse.device != device or tuple(lse.shape) != shape[:2]
                            or not lse.is_contiguous()):
        raise RuntimeError(f"lse must be a contiguous fp32 tensor {shape[:2]} on {device}")
    if ws is None:
        ws = workspace(step.workspace_bytes(cache.head_dim), device)
    _lib.call("nsmlp_paged_attention", ctypes.byref(cache._view), ctypes.byref(b._view), ctypes.byref(step._view), ptr(q),
              q.stride(0), q.stride(1), _DTYPES[q.dtype],
              1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), ptr(out), ptr(lse), ptr(ws), ws.numel(),
              stream_handle(device))
    return out
