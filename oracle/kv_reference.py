"""Plain restatements of the paged K/V cache for the tests: a step's plan with
loops, the codes in numpy (fp32 operations one by one, each rounded as
IEEE says, so codes and scales can be compared bit for bit) and the attention
in 64 bits with the masks written out."""
from __future__ import annotations

import numpy as np
import torch

SCALE_MIN = np.float32(2.0 ** -100)


class PlainBatch:
    """Requests' lengths, block lists and free blocks as Python lists."""

    def __init__(self, num_blocks, block, requests, max_blocks, free=None):
        self.block, self.max_blocks = block, max_blocks
        self.free = list(range(num_blocks)) if free is None else [int(b) for b in free]
        self.blocks = [[] for _ in range(requests)]
        self.cached = [0] * requests
        self._next = None

    def plan(self, new, total, max_new=0):
        B = self.block
        asked, taken, refused = 0, 0, 0
        slots, kv_len, q_start, blocks, nxt = [], [], [0], [], []
        for r, n in enumerate(new):
            have, tot = -(-self.cached[r] // B), -(-(self.cached[r] + n) // B)
            ok = tot <= self.max_blocks and (max_new == 0 or n <= max_new)
            need = tot - have if ok else 0  # what is refused for its length asks for nothing
            if need:
                ok = ok and asked + need <= len(self.free)
                asked += need
            mine = list(self.blocks[r])
            if ok:
                mine += self.free[asked - need: asked]
                taken += need
            refused += (not ok) and n > 0
            for p in range(self.cached[r], self.cached[r] + n):
                slots.append(mine[p // B] * B + p % B if ok else -1)
            kv_len.append(self.cached[r] + n if ok else 0)
            nxt.append(self.cached[r] + n if ok else self.cached[r])
            q_start.append(q_start[-1] + n)
            blocks.append(mine)
        slots = (slots + [-1] * total)[:total]
        self._next = (blocks, nxt, taken)
        return {"slots": slots, "kv_len": kv_len, "q_start": q_start, "blocks": blocks, "refused": refused,
                "free": len(self.free) - taken}

    def commit(self, finished=()):
        if self._next is not None:
            self.blocks, self.cached, taken = self._next
            self.free = self.free[taken:]
            self._next = None
        for r in finished:
            self.free += self.blocks[r]
            self.blocks[r], self.cached[r] = [], 0


def _e4m3(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.float8_e4m3fn).to(torch.float32).numpy()


def encode(x: np.ndarray, fmt: str) -> np.ndarray:
    """fp32 value / scale -> the value of its code (0 where it is not finite)."""
    x = np.where(np.isfinite(x), x, np.float32(0)).astype(np.float32)
    return np.clip(np.rint(x), -127, 127).astype(np.float32) if fmt == "int8" else _e4m3(np.clip(x, -448, 448))


def scale_of(amax: np.float32, fmt: str) -> np.float32:
    if not np.isfinite(amax):
        return np.float32(np.nan)
    if fmt == "int8":
        s = np.float32(amax) * (np.float32(1) / np.float32(127))
    elif amax == 0:
        s = np.float32(0)
    else:
        e = int(np.ceil(np.log2(np.float64(amax) / 448.0) - 1e-9))
        s = np.float32(2.0) ** np.float32(max(e, -140))
        while np.float64(amax) > 448.0 * np.float64(s):
            s = np.float32(s * 2)
    return max(np.float32(s), SCALE_MIN)


GRID4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode4(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Rows [..., dim] -> (values of their e2m1 codes, scale of each 32 dims), by trying every exponent and every code."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    most = np.abs(g).max(-1)
    scale = np.full(most.shape, 2.0 ** 13)
    for e in range(12, -24, -1):
        scale = np.where(most <= 6.0 * 2.0 ** e, 2.0 ** e, scale)
    away = np.abs(np.minimum(np.abs(g / scale[..., None]), 8.0)[..., None] - GRID4)
    # the nearest; of two as near the even one
    code = np.argmin(away + np.where(np.arange(8) % 2, 2.0 ** -40, 0.0), -1)
    return (np.sign(g) * GRID4[code]).reshape(x.shape).astype(np.float32), scale.astype(np.float32)


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """Rows [tokens, heads, dim] in fp16 or bf16 under cos, sin [tokens, dim / 2] in fp32: 64 bits, then fp32, then the type."""
    d = x.double()
    half = x.shape[-1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = torch.empty_like(d)
    at = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, half), slice(half, None))
    out[..., at[0]] = d[..., at[0]] * c - d[..., at[1]] * s
    out[..., at[1]] = d[..., at[1]] * c + d[..., at[0]] * s
    return out.float().to(x.dtype)


class PlainCache:
    """codes (as fp32 values) [blocks, heads, 2, block, dim], scale [blocks, heads, 2] (e2m1: [blocks, heads, 2, block, dim / 32])."""

    def __init__(self, blocks, heads, dim, block, fmt):
        self.fmt, self.block = fmt, block
        self.codes = np.zeros((blocks, heads, 2, block, dim), np.float32)
        self.scale = np.zeros((blocks, heads, 2) + ((block, dim // 32) if fmt == "e2m1" else ()), np.float32)

    def append(self, k: np.ndarray, v: np.ndarray, slots) -> None:
        """k, v [tokens, heads, dim] fp32; a block's tokens one after the other."""
        if self.fmt == "e2m1":
            for i, s in enumerate(int(s) for s in slots):
                for h in range(k.shape[1] if s >= 0 else 0):
                    finite = np.isfinite(k[i, h]).all() and np.isfinite(v[i, h]).all()
                    for which, x in ((0, k), (1, v)):
                        codes, scale = encode4(x[i, h]) if finite else (0.0, np.nan)
                        self.codes[s // self.block, h, which, s % self.block] = codes
                        self.scale[s // self.block, h, which, s % self.block] = scale
            return
        B, i, slots = self.block, 0, [int(s) for s in slots]
        while i < len(slots):
            if slots[i] < 0:
                i += 1
                continue
            n = 1
            while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] // B == slots[i] // B:
                n += 1
            b, off = slots[i] // B, slots[i] % B
            for which, x in ((0, k), (1, v)):
                for h in range(x.shape[1]):
                    rows = x[i: i + n, h].astype(np.float32)
                    old = np.float32(0) if off == 0 else self.scale[b, h, which]
                    amax = np.float32(np.abs(rows).max()) if np.isfinite(rows).all() else np.float32(np.inf)
                    need = scale_of(amax, self.fmt)
                    new = np.float32(np.nan) if np.isnan(need) or np.isnan(old) else max(old, need)
                    with np.errstate(invalid="ignore", over="ignore"):
                        if off and not new == old:
                            stored = self.codes[b, h, which, :off] * old
                            self.codes[b, h, which, :off] = encode(stored / new, self.fmt)
                        self.codes[b, h, which, off: off + n] = encode(rows / new, self.fmt)
                    self.scale[b, h, which] = new
            i += n

    def values(self, slots, which: int) -> np.ndarray:
        """fp32 values [tokens, heads, dim]: code * scale, rounded once."""
        s = np.asarray(slots, np.int64)
        if self.fmt == "e2m1":
            at = (s // self.block, slice(None), which, s % self.block)
            out = self.codes[at] * np.repeat(self.scale[at], 32, -1)
            out[s < 0] = 0
            return out
        out = self.codes[s // self.block, :, which, s % self.block] * self.scale[s // self.block][:, :, which, None]
        out[s < 0] = 0
        return out


def attention(q, keys, values, q_len, kv_len, scale):
    """One request in 64 bits: q [q_len, Hq, D], keys and values [kv_len, H, D]
    -> (out, lse, spread): spread = sum_j p_j |v_j|, what a weight's relative error is measured against."""
    q, keys, values = (torch.as_tensor(t).double() for t in (q, keys, values))
    G = q.shape[1] // keys.shape[1]
    out, lse, spread = torch.zeros_like(q), torch.full(q.shape[:2], -np.inf, dtype=torch.float64), torch.zeros_like(q)
    for i in range(q_len):
        n = kv_len - q_len + i + 1
        if n <= 0:
            continue
        for h in range(q.shape[1]):
            s = keys[:n, h // G] @ q[i, h] * scale
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[i, h] = p @ values[:n, h // G]
            spread[i, h] = p @ values[:n, h // G].abs()
    return out, lse, spread
