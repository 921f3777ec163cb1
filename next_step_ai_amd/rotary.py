"""Angles of a rotary position encoding, for ``KvCache.append_rotated``.

The frequencies are base^(-2 i / head_dim), i < head_dim / 2, or the caller's;
``scaling`` stretches them as a model's configuration says ("linear": all by
``factor``; "llama3": waves longer than original_max_position_embeddings /
low_freq_factor by ``factor``, those shorter than it over high_freq_factor not
at all, those between by a share of it).  Whole heads are turned.  Scalings that
multiply cos and sin by a factor take their own frequencies and, as q and k have
the factor each, its square times the softmax scale.  The reference leaves the encoding to
its model library (RT:5927-7142 call it with precomputed cos and sin).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._runtime import ptr, require_device

__all__ = ["Rotary", "rotary_frequencies"]


def rotary_frequencies(head_dim: int, base: float = 10000.0, scaling: dict | None = None) -> torch.Tensor:
    """The frequencies [head_dim / 2] in fp64, on the host."""
    if not (base > 0.0 and math.isfinite(base)):
        raise RuntimeError(f"base {base} must be positive and finite")
    f = float(base) ** -(torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    if scaling is None:
        return f
    # (what a configuration may say next to the scaling: left out, it would turn all rows by wrong angles)
    if scaling.get("partial_rotary_factor") not in (None, 1):
        raise RuntimeError(f"partial_rotary_factor {scaling['partial_rotary_factor']}: a part of a head's dims is not offered")
    if scaling.get("rope_theta") not in (None, base):
        raise RuntimeError(f"the scaling's rope_theta {scaling['rope_theta']} is not the base {base}")
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default"):
        return f
    if kind not in ("linear", "llama3"):
        raise RuntimeError(f"scaling of type {kind!r} is not offered: give its frequencies instead, and where it multiplies cos and "
                           "sin by a factor, the attention a softmax scale times that factor's square")
    need = ["factor"] if kind == "linear" else ["factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"]
    missing = [k for k in need if k not in scaling]
    if missing:
        raise RuntimeError(f"scaling of type {kind!r} needs {', '.join(missing)}")
    factor = float(scaling["factor"])
    if not factor >= 1.0:
        raise RuntimeError(f"scaling factor {factor} must be at least 1")
    if kind == "linear":
        return f / factor
    low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
    if not high > low:
        raise RuntimeError(f"high_freq_factor {high} must be above low_freq_factor {low}")
    span = float(scaling["original_max_position_embeddings"])
    share = ((span * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (1 - share) * f / factor + share * f


class Rotary:
    """cos and sin of ``positions`` positions: ``table`` [positions, head_dim /
    2, 2] fp32, from angles in fp64.  ``interleaved``: frequency i turns dims 2 i
    and 2 i + 1, else i and i + head_dim / 2.  ``frequencies`` [head_dim / 2]
    in place of those of ``base`` and ``scaling``."""

    def __init__(self, head_dim: int, positions: int, *, base: float = 10000.0, scaling: dict | None = None,
                 frequencies: torch.Tensor | None = None, interleaved: bool = False, device=None):
        if head_dim not in (64, 128):
            raise RuntimeError(f"head_dim must be 64 or 128, got {head_dim}")
        if not 1 <= positions <= 1 << 29:
            raise RuntimeError(f"positions must be in [1, 2^29], got {positions}")
        f = rotary_frequencies(head_dim, base, scaling) if frequencies is None else frequencies.double().reshape(-1)
        if f.numel() != head_dim // 2:
            raise RuntimeError(f"{head_dim // 2} frequencies expected, got {f.numel()}")
        self.device = require_device(torch.empty(0, device="cuda" if device is None else device), "rotary table")
        self.head_dim, self.positions, self.interleaved = int(head_dim), int(positions), bool(interleaved)
        self.table = torch.empty(self.positions, head_dim // 2, 2, dtype=torch.float32, device=self.device)
        f = f.to(self.device)
        for p in range(0, self.positions, 1 << 18):  # (fp64 angles of so many at a time)
            part = self.table[p: p + (1 << 18)]
            a = torch.arange(p, p + part.shape[0], dtype=torch.float64, device=self.device)[:, None] * f
            part[:, :, 0], part[:, :, 1] = a.cos(), a.sin()
        self._view = _lib.RotaryView(positions=self.positions, head_dim=self.head_dim, interleaved=int(self.interleaved),
                                     table=ptr(self.table))
        self._ref = ctypes.byref(self._view)
