"""Rotary positions in the forms language models use: half or interleaved pairs, all of a head or its first elements,
frequencies scaled for contexts longer than those trained on.

The angles are a table, computed once in 64 bits and kept on the device; the rotation itself is ``nkv_rotary``.  (The
3-D rotation of the reference's video models, with its own tables, is ``attention.RopeTable``.)
"""
from __future__ import annotations

import math

import torch

from . import ops


def frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Frequencies f64 [rotary_dim/2] and the factor on the table's entries.

    ``scaling``: None, or a dictionary with ``kind`` and ``factor``:
      linear  positions are divided by ``factor``
      base    the base grows so that the slowest frequency slows down by ``factor`` and the fastest stays
      blend   with ``trained`` positions: frequencies that turn fewer than ``low`` (1) times over them are divided by
              ``factor``, those that turn more than ``high`` (32) times stay, between the two a linear blend; entries are
              multiplied by ``gain`` (0.1 ln(factor) + 1), which sharpens the softmax of longer contexts
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even; got {rotary_dim}")
    exponent = torch.arange(rotary_dim // 2, dtype=torch.float64) * (2.0 / rotary_dim)
    if scaling is None:
        return base ** -exponent, 1.0
    kind, factor = scaling.get("kind"), float(scaling.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError(f"scaling factor must be at least 1; got {factor}")
    if kind == "linear":
        return base ** -exponent / factor, 1.0
    if kind == "base":
        if rotary_dim < 4:
            raise ValueError("scaling 'base' needs at least two frequencies")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -exponent, 1.0
    if kind == "blend":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 32.0))
        if not 0 < low < high:
            raise ValueError(f"scaling 'blend' needs 0 < low < high; got {low} and {high}")
        freq = base ** -exponent
        kept = ((float(scaling["trained"]) * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return freq / factor * (1 - kept) + freq * kept, float(scaling.get("gain", 0.1 * math.log(factor) + 1))
    raise ValueError(f"unknown scaling {kind!r}")


class Rotary:
    """Rotation of heads of ``head_dim`` elements at positions 0 .. rows - 1."""

    def __init__(self, head_dim: int, rows: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 layout: str = "half", scaling: dict | None = None, device="cuda"):
        freq, gain = frequencies(head_dim if rotary_dim is None else rotary_dim, base=base, scaling=scaling)
        angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
        table = (torch.stack([angle.cos(), angle.sin()], -1) * gain).to(torch.float32)
        self._take(table.to(device), head_dim, layout)

    @classmethod
    def over(cls, table: torch.Tensor, *, head_dim: int, layout: str = "half") -> "Rotary":
        """A rotation by a table that exists already: f32 [rows, rotary_dim/2, 2], cosine and sine."""
        self = cls.__new__(cls)
        self._take(table, head_dim, layout)
        return self

    def _take(self, table: torch.Tensor, head_dim: int, layout: str) -> None:
        if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous():
            raise ValueError("rotation table must be contiguous float32 [rows, rotary_dim/2, 2]")
        if not 0 < 2 * table.shape[1] <= head_dim:
            raise ValueError(f"the table turns {2 * table.shape[1]} elements of heads of {head_dim}")
        if layout not in ops._LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(ops._LAYOUTS)}; got {layout!r}")
        self.table, self.head_dim, self.layout = table, int(head_dim), layout

    @property
    def rotary_dim(self) -> int:
        return 2 * self.table.shape[1]

    @property
    def rows(self) -> int:
        return self.table.shape[0]

    def apply(self, q: torch.Tensor, k: torch.Tensor | None = None, *, positions: torch.Tensor, transposed: bool = False):
        """q (and k) [batch, tokens, heads, head_dim] rotated by positions i32 [batch, tokens], one launch for both.
        ``transposed``: the direction in which a gradient goes back.  A position outside the table gives NaN."""
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"heads are {q.shape[-1]} wide, the rotation is for {self.head_dim}")
        return ops.rotary(q, k, self.table, positions, layout=self.layout, transposed=transposed)
