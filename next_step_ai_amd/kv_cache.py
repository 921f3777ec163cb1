"""Paged K/V cache in 8 or 4 bits and the attention that reads it: the
attention side of the decoder layers whose MLPs the rest of the package runs.

    cache = KvCache(num_blocks, kv_heads, head_dim)              # one per layer
    batch = KvBatch(num_blocks, 16, max_requests=R, max_blocks=W, q_heads=Hq, kv_heads=H, head_dim=D)
    step = batch.plan(new_tokens, total, max_new=n)              # once per step, for every layer
    cache.append(k, v, step.slots)                               # per layer, or with a rotary encoding:
    q = cache.append_rotated(k, v, step.slots, step.positions, rotary, q=q)
    out = paged_attention(q, cache, step)                        # [total, Hq, D]
    batch.commit(finished)                                       # once per step

``KvBatch`` keeps the requests' lengths, block tables and free blocks on the
device; a step's plan is one kernel, and no call synchronises.  ``KvCache``
holds a layer's K and V codes with one scale per (block, head) for each in 8
bits, one per 32 dims of a token in 4 bits; the formats are described in
``nsmlp.h``.  The reference has no such cache: its
attention and K/V cache are torch code in ``streaming_llama_runtime.py``
(RT:5927-7142).  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._runtime import current_device, ptr, require_device, stream_handle, workspace
from .rotary import Rotary

__all__ = ["KvCache", "KvBatch", "KvStep", "paged_attention"]

_FORMATS = {"int8": _lib.NSMLP_KV_INT8, "e4m3": _lib.NSMLP_KV_E4M3, "e2m1": _lib.NSMLP_KV_E2M1}
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


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory between two tensors' first and last elements meets."""
    def span(t: torch.Tensor) -> tuple[int, int]:
        ends = [(n - 1) * s for n, s in zip(t.shape, t.stride())]
        first = t.data_ptr() + t.element_size() * sum(e for e in ends if e < 0)
        return first, t.data_ptr() + t.element_size() * (sum(e for e in ends if e > 0) + 1)

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _meets_itself(n: int, row: int, heads: int, head: int, dim: int) -> bool:
    """Whether rows [n, heads, dim] of these strides have memory in common."""
    inner, outer = ((heads, head), (n, row)) if head <= row else ((n, row), (heads, head))
    if inner[0] > 1 and inner[1] < dim:
        return True
    return outer[0] > 1 and outer[1] < (max(inner[0], 1) - 1) * inner[1] + dim


def _slots(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int64 or t.dim() != 1 or t.device != device:
        raise RuntimeError(f"slots must be an int64 [tokens] tensor on {device}")
    return t.contiguous()


class KvCache:
    """A layer's K and V: ``num_blocks`` blocks of ``block_tokens`` (16, 32 or
    64) tokens, ``fmt`` "int8", "e4m3" or, in 4 bits, "e2m1", ``head_dim`` 64 or
    128.  ``data`` holds the codes, ``scale`` the (block, head)s' scales (None in
    4 bits, where they stand among the codes)."""

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
        self._index = self.device.index
        self.num_blocks, self.kv_heads, self.head_dim = int(num_blocks), int(kv_heads), int(head_dim)
        self.block_tokens, self.fmt = int(block_tokens), fmt
        if fmt == "e2m1":
            self.data = torch.zeros(num_blocks, kv_heads, block_tokens * head_dim * 17 // 16, dtype=torch.uint8, device=self.device)
            self.scale = None
        else:
            self.data = torch.zeros(num_blocks, kv_heads, 2, block_tokens * head_dim, dtype=torch.uint8, device=self.device)
            self.scale = torch.zeros(num_blocks, kv_heads, 2, dtype=torch.float32, device=self.device)
        # (new tensors from one of their type take 1.2 us; torch.empty with a dtype and a device takes 1.8)
        self._like = {t: torch.empty(0, dtype=t, device=self.device) for t in _DTYPES}
        self._view = _lib.KvCacheView(num_blocks=self.num_blocks, kv_heads=self.kv_heads, head_dim=self.head_dim,
                                      block_tokens=self.block_tokens, format=_FORMATS[fmt], data=ptr(self.data),
                                      scale=ptr(self.scale))
        self._ref = ctypes.byref(self._view)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store the rows ``k``, ``v`` [tokens, kv_heads, head_dim] at ``slots``
        (a plan's: a block's tokens stand next to each other, in order, none
        twice; a slot of -1 stores nothing).  Where the new rows exceed a block's
        scale in 8 bits its stored codes are rewritten under the larger one."""
        if current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.append(k, v, slots)
        k, kp, k_row, k_head = _rows(k, "k", self.kv_heads, self.head_dim, self.device)
        v, vp, v_row, v_head = _rows(v, "v", self.kv_heads, self.head_dim, self.device)
        slots = _slots(slots, self.device)
        n = slots.shape[0]
        self._same_length(k, v, n)
        _lib.call("nsmlp_kv_append", self._ref, kp, k_row, k_head, vp, v_row, v_head, _DTYPES[k.dtype], slots.data_ptr(), n,
                  stream_handle(self.device))

    def _same_length(self, k: torch.Tensor, v: torch.Tensor, n: int) -> None:
        if k.dtype != v.dtype or k.shape[0] != n or v.shape[0] != n:
            raise RuntimeError(f"k, v and slots must be of the same length and k and v of one dtype: got {tuple(k.shape)} "
                               f"{k.dtype}, {tuple(v.shape)} {v.dtype} and {n} slots")

    def append_rotated(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, rotary: Rotary,
                       *, q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """:meth:`append` with the rows of ``k`` turned by their ``positions``
        [tokens] (int32, a plan's) on the way, and those of ``q`` [tokens, heads,
        head_dim], which are returned in ``q_out`` (may be ``q`` itself).  What is
        stored is what ``append`` stores of rows turned in 64 bits and rounded to
        fp32 and to their type; ``k`` is not changed.  A position that is not in
        the table makes its rows NaN; a query row at a negative one (a token of no
        request) is left as it was in ``q_out`` (a new one holds anything there).
        A ``q_out`` that overlaps ``q`` otherwise, ``k`` or ``v`` is refused; slices
        of one projection or buffer do not."""
        if current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.append_rotated(k, v, slots, positions, rotary, q=q, q_out=q_out)
        k, kp, k_row, k_head = _rows(k, "k", self.kv_heads, self.head_dim, self.device)
        v, vp, v_row, v_head = _rows(v, "v", self.kv_heads, self.head_dim, self.device)
        slots = _slots(slots, self.device)
        n = slots.shape[0]
        self._same_length(k, v, n)
        if rotary.device != self.device or rotary.head_dim != self.head_dim:
            raise RuntimeError(f"the rotary table is for head_dim {rotary.head_dim} on {rotary.device}, the cache has "
                               f"{self.head_dim} on {self.device}")
        if positions.dtype != torch.int32 or positions.device != self.device or tuple(positions.shape) != (n,):
            raise RuntimeError(f"positions must be an int32 [{n}] tensor on {self.device}")
        positions = positions.contiguous()
        if q is None:
            if q_out is not None:
                raise RuntimeError("q_out without q")
            _lib.call("nsmlp_kv_append_rotated", self._ref, rotary._ref, kp, k_row, k_head, vp, v_row, v_head, _DTYPES[k.dtype],
                      slots.data_ptr(), positions.data_ptr(), n, None, 0, 0, 0, None, 0, 0, stream_handle(self.device))
            return None
        heads = q.shape[1] if q.dim() == 3 else 0
        rows, qp, q_row, q_head = _rows(q, "q", heads, self.head_dim, self.device)
        if rows.shape[0] != n or rows.dtype != k.dtype or heads < 1:
            raise RuntimeError(f"q must be [{n}, heads, {self.head_dim}] of k's dtype {k.dtype}, got {tuple(q.shape)} {q.dtype}")
        if q_out is None:
            q_out = rows.new_empty((n, heads, self.head_dim))
            op, o_row, o_head = q_out.data_ptr(), heads * self.head_dim, self.head_dim
        else:
            if q_out.dtype != rows.dtype or q_out.shape != q.shape:
                raise RuntimeError(f"q_out must be {tuple(q.shape)} {q.dtype}, got {tuple(q_out.shape)} {q_out.dtype}")
            out, op, o_row, o_head = _rows(q_out, "q_out", heads, self.head_dim, self.device)
            if out is not q_out or _meets_itself(n, o_row, heads, o_head, self.head_dim):
                raise RuntimeError("q_out must be 16-byte aligned with strides that are multiples of 8 elements, and no element twice")
        _lib.call("nsmlp_kv_append_rotated", self._ref, rotary._ref, kp, k_row, k_head, vp, v_row, v_head, _DTYPES[k.dtype],
                  slots.data_ptr(), positions.data_ptr(), n, qp, q_row, q_head, heads, op, o_row, o_head,
                  stream_handle(self.device))
        return q_out

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> dict[str, torch.Tensor]:
        """The stored rows at ``slots``: ``{"k": ..., "v": ...}`` of [tokens,
        kv_heads, head_dim] in ``dtype``; zeros for a slot of -1."""
        if current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.read(slots, dtype)
        if dtype not in _DTYPES:
            raise RuntimeError(f"dtype must be fp16 or bf16, got {dtype}")
        slots = _slots(slots, self.device)
        n = slots.shape[0]
        shape = (n, self.kv_heads, self.head_dim)
        like = self._like[dtype]
        k, v = like.new_empty(shape), like.new_empty(shape)
        _lib.call("nsmlp_kv_read", self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _DTYPES[dtype],
                  stream_handle(self.device))
        return {"k": k, "v": v}


class _StepLayout:
    """Sizes of a step's buffers, which depend on its total and max_new alone."""

    __slots__ = ("ints", "positions_at", "sizes", "offsets", "schedule_bytes", "ws_bytes")

    def __init__(self, batch: "KvBatch", total: int, max_new: int):
        self.schedule_bytes = int(_lib.lib().nsmlp_kv_schedule_bytes(batch._ref, total, max_new))
        if self.schedule_bytes == 0:
            raise RuntimeError(f"nsmlp_kv_schedule_bytes: {_lib.last_error()}")
        R = batch.requests
        self.ints = (3 * R + 5 + 3) // 4 * 4
        self.positions_at = self.ints + self.schedule_bytes // 4
        self.sizes = [R + 1, R, R, 4, self.positions_at - 3 * R - 5 + total]
        self.offsets = tuple(4 * i for i in (R + 1, 2 * R + 1, 3 * R + 1, self.ints, self.positions_at))
        self.ws_bytes: dict[int, int] = {}


class KvStep:
    """A planned step: ``slots`` [total] int64 (-1: none), ``positions``
    [total] (how many of its request's tokens stand before each; -1: none),
    ``q_start`` [requests + 1], ``kv_len`` [requests], ``info`` [4] = (ring head, free
    blocks, refused requests, sum of new tokens) after it, ``table`` the batch's
    block table.  ``info`` and the others are device tensors: reading them
    waits for the stream.  ``planned``: whether a plan has written them."""

    __slots__ = ("batch", "total", "max_new", "slots", "planned", "_buf", "_layout", "_view", "_ref", "_split", "_positions")

    def __init__(self, batch: "KvBatch", total: int, max_new: int):
        lay = batch._layout(total, max_new)
        self.batch, self.total, self.max_new, self._layout = batch, total, max_new, lay
        self.slots = batch._slot.new_empty(total)  # (1.2 us; torch.empty with a dtype and a device takes 1.7)
        # q_start, kv_len, next and info, then the schedule at the next 16 bytes, then positions
        self._buf = batch.state.new_empty(lay.positions_at + total)
        base = self._buf.data_ptr()
        kv_len, following, info, schedule, positions = lay.offsets
        self._view = _lib.KvStepView(total, max_new, self.slots.data_ptr(), base, base + kv_len, base + following, base + info,
                                     base + schedule, lay.schedule_bytes, base + positions)
        self._ref = ctypes.byref(self._view)
        self._split = self._positions = None
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
    def positions(self) -> torch.Tensor:
        if self._positions is None:  # (a view of its own: steps without a rotation do not make it)
            self._positions = self._buf[self._layout.positions_at:]
        return self._positions

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
        self._index = self.device.index
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
        if current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.plan(new_tokens, total, max_new=max_new, step=step)
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
        if current_device() != self._index:
            with torch.cuda.device(self.device):
                return self.commit(finished)
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
    1/sqrt(head_dim).  Returns ``out`` [total, q_heads, head_dim], contiguous,
    which may be ``q`` itself and overlaps it in no other way; ``lse``
    ([total, q_heads] fp32) receives the log of the softmax sums.  ``ws``: a
    uint8 workspace of ``step.workspace_bytes(head_dim)`` that
    ``nsmlp_workspace_init`` has cleared, in place of the stream's own."""
    b, device, dim = step.batch, cache.device, cache.head_dim
    if b.device != device:
        raise RuntimeError(f"the cache is on {device} and the batch on {b.device}")
    if current_device() != cache._index:
        with torch.cuda.device(device):
            return paged_attention(q, cache, step, scale=scale, out=out, lse=lse, ws=ws)
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
    elif total and _overlap(q, out) and not (out.data_ptr() == qp and q.is_contiguous()):
        # (in place: a row of out is written when all that read the same row of q have done so)
        raise RuntimeError("out overlaps q: it must be q's own memory, both contiguous, or lie apart from it")
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
