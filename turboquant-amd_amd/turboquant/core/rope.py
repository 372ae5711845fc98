"""Frequencies of rotary positions, on the host: turns per position of each pair, and the rows' magnitude.

kernels.rotation.apply_rope takes the result.  Scalings for contexts longer than the trained one, by
`factor` (new length / trained length):

  "linear"    every frequency divided by factor (positions interpolated)
  "base"      the base theta raised to theta * factor^(d / (d - 2)): the fastest pair keeps its frequency,
              the slowest is divided by factor
  "by_parts"  pairs that turn at least `fast` times over the trained length keep their frequency, those that turn
              at most `slow` times are divided by factor, those between are blended; rows are scaled by
              0.1 ln(factor) + 1.  blend="turns": linearly in the number of turns, as the method was published;
              blend="index": linearly in the pair's index, between the indices of `fast` turns, rounded down, and
              of `slow` turns, rounded up.  At factor 4 the two differ by up to 43 % in between; released checkpoints
              with this scaling were commonly trained with "index": take what the checkpoint's own code does
"""

from __future__ import annotations

import math
from typing import Optional

import torch


def rope_turns(rotary_dim: int = 128, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               trained_length: int = 32768, fast: float = 32.0, slow: float = 1.0,
               device=None, blend: str = "turns") -> tuple[torch.Tensor, float]:
    """(turns float64 [rotary_dim / 2], magnitude): pair i turns theta^(-2i / rotary_dim) / (2 pi) per position,
    scaled as named above."""
    if rotary_dim < 2 or rotary_dim > 128 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and in 2..128, got {rotary_dim}")
    if not theta > 0 or not factor > 0:
        raise ValueError("theta and factor must be positive")
    if scaling not in (None, "linear", "base", "by_parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'by_parts', got {scaling!r}")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling='base' needs rotary_dim > 2")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    turns = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim) / (2 * math.pi)
    magnitude = 1.0
    if scaling == "linear":
        turns = turns / factor
    elif scaling == "by_parts":
        if not fast > slow or trained_length <= 0:
            raise ValueError("scaling='by_parts' needs fast > slow and a positive trained_length")
        if blend not in ("turns", "index"):
            raise ValueError(f"blend must be 'turns' or 'index', got {blend!r}")
        n = turns * trained_length
        if blend == "turns":
            keep = ((n - slow) / (fast - slow)).clamp(0.0, 1.0)
        else:
            if not theta > 1 or not slow > 0:
                raise ValueError("blend='index' needs theta > 1 and slow > 0")
            # pair i turns m times where theta^(-2i / rotary_dim) trained_length / (2 pi) = m
            first, last = (0.5 * rotary_dim * math.log(trained_length / (2 * math.pi * m)) / math.log(theta) for m in (fast, slow))
            first, last = max(math.floor(first), 0), min(math.ceil(last), rotary_dim - 1)
            i = torch.arange(rotary_dim // 2, dtype=torch.float64)
            keep = ((last - i) / (last - first)).clamp(0.0, 1.0) if last > first else (i <= first).double()
            keep = torch.where(n > slow, keep, 0.0)
        turns = turns / factor * (1 - keep) + turns * keep
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return turns.to(device), magnitude
