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

import torch

from . import _lib
from ._runtime import ptr, require_device, stream_handle, workspace

__all__ = ["KvCache", "KvBatch", "KvStep", "paged_attention"]

_FORMATS = {"int8": _lib.NSMLP_KV_INT8, "e4m3": _lib.NSMLP_KV_E4M3}
_DTYPES = {torch.float16: _lib.NSMLP_DTYPE_F16, torch.bfloat16: _lib.NSMLP_DTYPE_BF16}


def _device(device) -> torch.device:
    return require_device(torch.empty(0, device="cuda" if device is None else device), "cache")


def _rows(t: torch.Tensor, what: str, heads: int, dim: int, device: torch.device) -> tuple[torch.Tensor, int, int, int]:
    """(tensor, address, row and head stride) of [tokens, heads, dim] in fp16 or
    bf16 that the kernels can read in 16-byte pieces; a copy where the strides
    do not allow it."""
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{what} must be fp16 or bf16, got {t.dtype}")
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise RuntimeError(f"{what} must be [tokens, {heads}, {dim}], got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{what} must be a GPU tensor on {device}, got {t.device}")
    row, head, one = t.stride()
    # (a dimension of one element may have any stride, and a copy keeps it)
    if t.shape[0] <= 1:
        row = heads * dim
    if heads == 1:
        head = dim
    p = t.data_ptr()
    if one != 1 or row % 8 or head % 8 or p % 16:
        t = t.contiguous()
        t = t if t.data_ptr() % 16 == 0 else t.clone()
        row, head = heads * dim, dim
        p = t.data_ptr()
    return t, p, row, head


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
        self._ref = ctypes.byref(self._view)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store the rows ``k``, ``v`` [tokens, kv_heads, head_dim] at ``slots``
        (a plan's: a block's tokens stand next to each other, in order; a slot
        of -1 stores nothing).  Where the new rows exceed a block's scale its
        stored codes are rewritten under the larger one."""
        k, kp, k_row, k_head = _rows(k, "k", self.kv_heads, self.head_dim, self.device)
        v, vp, v_row, v_head = _rows(v, "v", self.kv_heads, self.head_dim, self.device)
        slots = _slots(slots, self.device)
        n = slots.shape[0]
        if k.dtype != v.dtype or k.shape[0] != n or v.shape[0] != n:
            raise RuntimeError(f"k, v and slots must be of the same length and k and v of one dtype: got {tuple(k.shape)} "
                               f"{k.dtype}, {tuple(v.shape)} {v.dtype} and {n} slots")
        _lib.call("nsmlp_kv_append", self._ref, kp, k_row, k_head, vp, v_row, v_head, _DTYPES[k.dtype], slots.data_ptr(), n,
                  stream_handle(self.device))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> dict[str, torch.Tensor]:
        """The stored rows at ``slots``: ``{"k": ..., "v": ...}`` of [tokens,
        kv_heads, head_dim] in ``dtype``; zeros for a slot of -1."""
        if dtype not in _DTYPES:
            raise RuntimeError(f"dtype must be fp16 or bf16, got {dtype}")
        slots = _slots(slots, self.device)
        n = slots.shape[0]
        shape = (n, self.kv_heads, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        _lib.call("nsmlp_kv_read", self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _DTYPES[dtype],
                  stream_handle(self.device))
        return {"k": k, "v": v}


class _StepLayout:
    """Sizes of a step's buffers, which depend on its total and max_new alone."""

    __slots__ = ("ints", "sizes", "schedule_bytes", "ws_bytes")

    def __init__(self, batch: "KvBatch", total: int, max_new: int):
        self.schedule_bytes = int(_lib.lib().nsmlp_kv_schedule_bytes(batch._ref, total, max_new))
        if self.schedule_bytes == 0:
            raise RuntimeError(f"nsmlp_kv_schedule_bytes: {_lib.last_error()}")
        R = batch.requests
        self.ints = (3 * R + 5 + 3) // 4 * 4
        self.sizes = [R + 1, R, R, 4, self.ints - 3 * R - 5 + self.schedule_bytes // 4]
        self.ws_bytes: dict[int, int] = {}


class KvStep:
    """A planned step: ``slots`` [total] int64 (-1: none), ``q_start``
    [requests + 1], ``kv_len`` [requests], ``info`` [4] = (ring head, free
    blocks, refused requests, sum of new tokens) after it, ``table`` the batch's
    block table.  ``info`` and the others are device tensors: reading them
    waits for the stream.  ``planned``: whether a plan has written them."""

    __slots__ = ("batch", "total", "max_new", "slots", "planned", "_buf", "_layout", "_view", "_ref", "_split")

    def __init__(self, batch: "KvBatch", total: int, max_new: int):
        lay = batch._layout(total, max_new)
        self.batch, self.total, self.max_new, self._layout = batch, total, max_new, lay
        self.slots = batch._slot.new_empty(total)  # (1.2 us; torch.empty with a dtype and a device takes 1.7)
        # q_start, kv_len, next and info, then the schedule at the next 16 bytes
        self._buf = batch.state.new_empty(lay.ints + lay.schedule_bytes // 4)
        base, R = self._buf.data_ptr(), batch.requests
        self._view = _lib.KvStepView(total, max_new, self.slots.data_ptr(), base, base + 4 * (R + 1), base + 4 * (2 * R + 1),
                                     base + 4 * (3 * R + 1), base + 4 * lay.ints, lay.schedule_bytes)
        self._ref = ctypes.byref(self._view)
        self._split = None
        self.planned = False

    def _part(self, i: int) -> torch.Tensor:
        if self._split is None:  # one split takes half as long as three views
            self._split = self._buf.split_with_sizes(self._layout.sizes)
        return self._split[i]

    @property
    def q_start(self) -> torch.Tensor:
        return self._part(0)

    @property
    def kv_len(self) -> torch.Tensor:
        return self._part(1)

    @property
    def info(self) -> torch.Tensor:
        return self._part(3)

    @property
    def table(self) -> torch.Tensor:
        return self.batch.table

    def workspace_bytes(self, head_dim: int) -> int:
        n = self._layout.ws_bytes.get(head_dim)
        if n is None:
            n = int(_lib.lib().nsmlp_paged_attention_workspace_bytes(self.batch._ref, self.total, self.max_new, head_dim))
            self._layout.ws_bytes[head_dim] = n
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
        self._slot = torch.empty(0, dtype=torch.int64, device=self.device)
        self._view = _lib.KvBatchView(requests=self.requests, max_blocks=self.max_blocks, num_blocks=self.num_blocks,
                                      block_tokens=self.block_tokens, q_heads=self.q_heads, kv_heads=self.kv_heads,
                                      cached=ptr(self.cached), table=ptr(self.table), ring=ptr(self.ring),
                                      state=ptr(self.state))
        self._ref = ctypes.byref(self._view)
        self._layouts: dict[tuple[int, int], _StepLayout] = {}
        self._layout(1, 0)  # checks the arguments
        self._step: KvStep | None = None

    def _layout(self, total: int, max_new: int) -> _StepLayout:
        lay = self._layouts.get((total, max_new))
        if lay is None:
            if len(self._layouts) >= 1024:
                self._layouts.clear()
            lay = self._layouts[(total, max_new)] = _StepLayout(self, total, max_new)
        return lay

    def plan(self, new_tokens: torch.Tensor, total: int, *, max_new: int = 0, step: KvStep | None = None) -> KvStep:
        """Place the step's tokens: ``new_tokens`` [requests] int32 on the
        device (0 for a request that waits), ``total`` their sum, ``max_new``
        the most of one request where the caller knows it (it decides which
        kernels the attention launches).  Lengths and free blocks stay as they
        are until :meth:`commit`; a plan that is not committed can be made
        again (with other ``new_tokens``, requests after the first whose need
        of blocks changes get other ones).  ``step``: an earlier step of the same ``total`` and ``max_new``
        whose buffers are written again (a captured graph's)."""
        total, max_new = int(total), int(max_new)
        if new_tokens.dtype != torch.int32 or new_tokens.device != self.device or new_tokens.numel() != self.requests \
                or not new_tokens.is_contiguous():
            raise RuntimeError(f"new_tokens must be a contiguous int32 [{self.requests}] tensor on {self.device}")
        if step is None:
            step = KvStep(self, total, max_new)
        elif step.batch is not self or step.total != total or step.max_new != max_new:
            raise RuntimeError("the step to plan into belongs to another batch, total or max_new")
        _lib.call("nsmlp_kv_plan", self._ref, new_tokens.data_ptr(), step._ref, stream_handle(self.device))
        step.planned = True
        self._step = step
        return step

    def commit(self, finished: torch.Tensor | None = None) -> None:
        """Make the last plan's lengths (all of its new tokens) the batch's, and end the requests with
        ``finished`` [requests] (int32, not 0): their blocks become free."""
        if finished is not None and (finished.dtype != torch.int32 or finished.device != self.device
                                     or int(finished.numel()) != self.requests or not finished.is_contiguous()):
            raise RuntimeError(f"finished must be a contiguous int32 [{self.requests}] tensor on {self.device}")
        st = self._step
        _lib.call("nsmlp_kv_commit", self._ref, None if st is None else st._ref, ptr(finished), stream_handle(self.device))
        self._step = None  # (a commit that fails can be made again)


def paged_attention(q: torch.Tensor, cache: KvCache, step: KvStep, *, scale: float | None = None,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    ws: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's queries ``q`` [total, q_heads, head_dim] (fp16 or
    bf16) over the cache, causal at the end of each request (its new tokens'
    K and V are appended before the call).  ``scale`` defaults to
    1/sqrt(head_dim).  Returns ``out`` [total, q_heads, head_dim]; ``lse``
    ([total, q_heads] fp32) receives the log of the softmax sums.  ``ws``: a
    uint8 workspace of ``step.workspace_bytes(head_dim)`` that
    ``nsmlp_workspace_init`` has cleared, in place of the stream's own."""
    b, device, dim = step.batch, cache.device, cache.head_dim
    if b.device != device:
        raise RuntimeError(f"the cache is on {device} and the batch on {b.device}")
    if not step.planned:  # its lists are what the memory held
        raise RuntimeError("the step has not been planned (KvBatch.plan)")
    total, heads = step.total, b.q_heads
    q, qp, q_row, q_head = _rows(q, "q", heads, dim, device)
    if q.shape[0] != total:
        raise RuntimeError(f"q holds {q.shape[0]} tokens, the step {total}")
    dtype = q.dtype
    if out is None:
        out = torch.empty((total, heads, dim), dtype=dtype, device=device)
    elif out.dtype != dtype or out.device != device or tuple(out.shape) != (total, heads, dim) or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise RuntimeError(f"out must be a contiguous, 16-byte aligned {dtype} tensor {(total, heads, dim)} on {device}")
    if lse is not None and (lse.dtype != torch.float32 or lse.device != device or tuple(lse.shape) != (total, heads)
                            or not lse.is_contiguous()):
        raise RuntimeError(f"lse must be a contiguous fp32 tensor {(total, heads)} on {device}")
    if ws is None:
        ws = workspace(step.workspace_bytes(dim), device)
    elif ws.device != device or not ws.is_contiguous():
        raise RuntimeError(f"ws must be a contiguous tensor on {device}, got one on {ws.device} with strides {ws.stride()}")
    _lib.call("nsmlp_paged_attention", cache._ref, b._ref, step._ref, qp, q_row, q_head, _DTYPES[dtype],
              dim ** -0.5 if scale is None else float(scale), out.data_ptr(), None if lse is None else lse.data_ptr(),
              ws.data_ptr(), ws.numel(), stream_handle(device))
    return out
