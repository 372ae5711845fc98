"""Step planning on the GPU: block tables, slots, positions and lengths from the requests' lengths.

plan_step gives a step's layers what they take - slot_mapping (compress_paged_kv, quantize_paged8_kv),
positions (apply_rope), query_start_loc, seq_lens and block_tables (PagedDecodeMetadata) - without a copy of
any length to the host, so a serving loop can run it inside a captured graph.  Free blocks live in a ring
on the device: ring int32 [num_blocks] and pool int32 [2] = (first, count), see new_pool.
"""

from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional

import torch

from turboquant import _lib

_PLAN = struct.Struct("@3Qq8Q2q4i")


@dataclass
class StepPlan:
    """What one engine step needs (all on the device)."""

    query_start_loc: torch.Tensor  # int32 [S + 1]: new tokens of the requests before
    seq_lens: torch.Tensor         # int32 [S]: lengths after the step
    positions: torch.Tensor        # int32 [num_tokens]; 0 behind the last token
    slot_mapping: torch.Tensor     # int64 [num_tokens]; -1 behind the last token and for refused requests
    pool: torch.Tensor             # int32 [2]: (first, count) of the ring after the step


def new_pool(num_blocks: int, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(ring, pool) with all num_blocks blocks free."""
    if num_blocks <= 0:
        raise ValueError("num_blocks must be positive")
    return (torch.arange(num_blocks, dtype=torch.int32, device=device),
            torch.tensor([0, num_blocks], dtype=torch.int32, device=device))


def plan_step(
    past_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    ring: torch.Tensor,
    pool: torch.Tensor,
    block_size: int,
    num_tokens: int,
    pool_out: Optional[torch.Tensor] = None,
    out: Optional[StepPlan] = None,
) -> StepPlan:
    """Plan one step of requests that hold past_lens [S] cached tokens and get new_lens [S] more (both int32).

    new_lens < 0 gives up the last -new_lens tokens of a request (-past_lens ends it).  In request
    order, blocks for new tokens are taken from the ring's front into block_tables [S, max_blocks] (in
    place) and given-up blocks go to the ring's end; blocks given up in a step are handed out from the next one on.
    A request that the ring cannot serve any more (the needs of the requests before it counted), or
    whose table is too narrow, is not extended: its seq_lens entry stays past_lens and its tokens get slot
    -1, so that the cache writes skip them (what attention gives for those tokens means nothing).  A block
    belongs to one request: blocks that tables share would be given up twice.  num_tokens: size of the token arrays, at least the
    sum of the positive new_lens.  pool_out: where the ring's new (first, count) goes (default: pool
    itself).  out: a StepPlan whose arrays are written instead of new ones; its seq_lens may be past_lens.
    """
    dev = _lib.require_gpu("plan_step", past_lens, new_lens, block_tables, ring, pool, pool_out)
    if not (past_lens.dtype == new_lens.dtype == block_tables.dtype == ring.dtype == pool.dtype == torch.int32):
        raise TypeError("past_lens, new_lens, block_tables, ring and pool must be int32")
    if past_lens.dim() != 1 or new_lens.shape != past_lens.shape:
        raise ValueError("past_lens and new_lens must be [S]")
    S = past_lens.shape[0]
    if block_tables.dim() != 2 or block_tables.shape[0] != S or (block_tables.stride(1) != 1 and block_tables.shape[1] > 1):
        raise ValueError("block_tables must be [S, max_blocks] with unit inner stride")
    if ring.dim() != 1 or not ring.numel() or not ring.is_contiguous():
        raise ValueError("ring must be [num_blocks], contiguous")
    pool_out = pool if pool_out is None else pool_out
    if pool.shape != (2,) or pool_out.shape != (2,) or pool_out.dtype != torch.int32 or not pool.is_contiguous() or \
            not pool_out.is_contiguous():
        raise ValueError("pool and pool_out must be int32 [2], contiguous")
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    past_lens, new_lens = past_lens.contiguous(), new_lens.contiguous()
    L = _lib.lib()
    need = L.tq_plan_step_workspace_bytes(S)
    if out is None:
        # one allocation for the workspace and the 32-bit arrays behind it
        w = need // 4
        buf = torch.empty(w + 2 * S + 1 + num_tokens, dtype=torch.int32, device=dev)
        _, start, lens, positions = buf.split((w, S + 1, S, num_tokens))
        out = StepPlan(start, lens, positions, torch.empty(num_tokens, dtype=torch.int64, device=dev), pool_out)
    else:
        buf = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        for t, shape, dt in ((out.query_start_loc, (S + 1,), torch.int32), (out.seq_lens, (S,), torch.int32),
                             (out.positions, (num_tokens,), torch.int32), (out.slot_mapping, (num_tokens,), torch.int64)):
            if t.shape != shape or t.dtype != dt or not t.is_contiguous() or t.device != dev:
                raise ValueError("out does not match the step's sizes, types or device")
        out.pool = pool_out
    args = _PLAN.pack(past_lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(),
                      block_tables.stride(0) if S > 1 else block_tables.shape[1], ring.data_ptr(), pool.data_ptr(),
                      pool_out.data_ptr(), out.seq_lens.data_ptr(), out.query_start_loc.data_ptr(), out.positions.data_ptr(),
                      out.slot_mapping.data_ptr(), buf.data_ptr(), need, num_tokens, S, block_tables.shape[1], ring.shape[0],
                      int(block_size))
    _lib.launch("tq_plan_step", dev, args)
    return out
