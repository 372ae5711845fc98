"""Frequencies of rotary positions, on the host: turns per position of each pair, and the rows' magnitude.

kernels.rotation.apply_rope takes the result.  Scalings for contexts longer than the trained one, by
`factor` (new length / trained length):

  "linear"    every frequency divided by factor (positions interpolated)
  "base"      the base theta raised to theta * factor^(d / (d - 2)): the fastest pair keeps its frequency,
              the slowest is divided by factor
  "by_parts"  pairs that turn at least `fast` times over the trained length keep their frequency, those that turn
              at most `slow` times are divided by factor, those between are blended linearly in the number
              of turns; rows are scaled by 0.1 ln(factor) + 1
"""

from __future__ import annotations

import math
from typing import Optional

import torch


def rope_turns(rotary_dim: int = 128, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               trained_length: int = 32768, fast: float = 32.0, slow: float = 1.0,
               device=None) -> tuple[torch.Tensor, float]:
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
        keep = ((turns * trained_length - slow) / (fast - slow)).clamp(0.0, 1.0)
        turns = turns / factor * (1 - keep) + turns * keep
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return turns.to(device), magnitude
