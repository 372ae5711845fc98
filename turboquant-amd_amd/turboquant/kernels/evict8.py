"""Accumulated attention weights and eviction: sessions whose 8-bit paged cache (kernels.paged8) stays bounded.

Every cached token has a number per KV head, the sum of the softmax weights it got: mass, float32 [num_blocks,
num_kv_heads, block_size], paged like the cache.  decode_paged8(..., mass=mass) adds a step's weights,
observe_paged8 those of a prompt's queries; new tokens start from 0 in either, so a recycled block needs no clearing, as long as
every token is new in one of them: prompts are observed (last=1 is enough), and a request that plan_step could not serve is
left out of the step, whose calls would take its last cached tokens for new ones.
evict_paged8 then cuts each long sequence to its first, its last and its heaviest tokens, in place, and its result
is what plan_step takes as new_lens to give the blocks behind them back:

    change = evict_paged8(k_cache, k_fmt, v_cache, v_fmt, mass, tables, lens, keep=4096, recent=1024, sinks=4)
    plan_step(lens, change, tables, ring, pool, block_size, 0)

Layers share block tables, so each of them evicts, with its own cache and mass and the same keep, before
the one plan_step.  That takes a model all of whose layers are 8-bit ones: a packed layer has no eviction, and would be left with its
first `keep` tokens.  A cached token's index is then less than its position: a caller adds what each sequence gave up (the
sums of -change, once for each of its new tokens) to the positions that plan_step returns before apply_rope.
"""

from __future__ import annotations

import struct
from typing import Optional

import torch

from turboquant import _lib
from turboquant.kernels.paged import PREFILL_CAUSAL
from turboquant.kernels.paged8 import (_ATTN, _REACH, _SCALE, Paged8Format, _check_cache, _check_mass, _check_pair, _check_window,
                                       _rows)


def allocate_mass(num_blocks: int, num_kv_heads: int, block_size: int, device=None) -> torch.Tensor:
    """Accumulated weights of a cache, all 0."""
    return torch.zeros(num_blocks, num_kv_heads, block_size, dtype=torch.float32, device=device)


def _check_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor) -> tuple[int, int, int]:
    """(sequences, blocks per sequence, row stride)."""
    if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.shape[0] != seq_lens.shape[0] or (
            block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [num_seqs, max_blocks] with unit inner stride and seq_lens [num_seqs]")
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    S, mb = block_tables.shape
    return S, mb, block_tables.stride(0) if S > 1 else mb


def _workspace(workspace: Optional[torch.Tensor], need: int, dev: torch.device) -> torch.Tensor:
    if workspace is None:
        # (a buffer of this call: of the current stream, and of the graph under capture)
        return torch.empty(need, dtype=torch.uint8, device=dev)
    if workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 256 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be {need} contiguous bytes on {dev}, 256-byte aligned")
    return workspace


def _bound(max_seq_len: Optional[int], blocks: int, block_size: int) -> int:
    """The tokens of a sequence that a call looks at."""
    cap = min(blocks * block_size, 0x7fff0000)
    return cap if max_seq_len is None else max(0, min(int(max_seq_len), cap))


def observe_paged8(
    q: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    k_cache: torch.Tensor,
    k_fmt: Paged8Format,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    mass: torch.Tensor,
    sm_scale: Optional[float] = None,
    last: Optional[int] = None,
    max_q_len: Optional[int] = None,
    max_seq_len: Optional[int] = None,
    window: Optional[int] = None,
    sinks: int = 0,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Add the softmax weights that prompts' queries give to the cached tokens to mass [num_blocks, Hkv, block_size], in place.

    q [T, Hq, 128], cu_seqlens_q, block_tables and seq_lens as in prefill_paged8 (causal), whose call stands beside this
    one.  Of each sequence's new tokens the last `last` (default: all) count as queries; a token's number grows by the weights
    of its KV head's query heads over them, and the new tokens start from 0, whatever their rows held.  Sequences
    without new tokens keep their numbers.  Weights are those of the whole row (all visible tokens), in fp32; f32 queries are
    carried in twice fp16's precision.  A query whose weights are not numbers adds nothing.  max_q_len: host-side bound of the query
    counts (default: T); max_seq_len: of seq_lens (default: the tables' capacity).  window, sinks: as in prefill_paged8.  Blocks
    must belong to one sequence.  Workspace: tq_kv8_observe_workspace_bytes(...).
    """
    dev = _lib.require_gpu("observe_paged8", q, cu_seqlens_q, k_cache, block_tables, seq_lens, mass, workspace)
    if q.dim() != 3 or q.shape[2] != 128:
        raise ValueError("q must be [T, Hq, 128]")
    S, mb, row = _check_tables(block_tables, seq_lens)
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] != S + 1:
        raise ValueError("cu_seqlens_q must be [num_seqs + 1]")
    if cu_seqlens_q.dtype != torch.int32:
        raise TypeError("cu_seqlens_q must be int32")
    kb, kh = _check_cache(k_cache, k_fmt, "observe_paged8")
    if k_fmt.layout != "keys":
        raise ValueError("observe_paged8 reads a K cache (layout='keys')")
    nb, hkv, _ = k_cache.shape
    T, hq, _ = q.shape
    if not hkv or hq % hkv:
        raise ValueError(f"num_q_heads {hq} must be a multiple of num_kv_heads {hkv}")
    if not nb:
        raise ValueError("the cache holds no blocks")
    ms = _check_mass(mass, nb, hkv, k_fmt.block_size)
    scale = _SCALE if sm_scale is None else float(sm_scale)
    if not abs(scale) < float("inf"):
        raise ValueError("sm_scale must be finite")
    last = T if last is None else int(last)
    if last < 1 and T:
        raise ValueError(f"last must be positive, got {last}")
    window, sinks = _check_window(window, sinks)
    mq = T if max_q_len is None else max(0, min(int(max_q_len), T))
    if not T or not hq or not mq:
        return mass
    last = min(last, mq)
    q, seq_lens, cu_seqlens_q = _rows(q), seq_lens.contiguous(), cu_seqlens_q.contiguous()
    code, cap = _lib.dtype_code(q), _bound(max_seq_len, mb, k_fmt.block_size)
    need = _lib.lib().tq_kv8_observe_workspace_bytes(S, mq, last, hq, hkv, code, cap)
    ws = _workspace(workspace, need, dev)
    qt, qh, _ = q.stride()
    args = _ATTN.pack(q.data_ptr(), 0, k_cache.data_ptr(), 0, block_tables.data_ptr(), seq_lens.data_ptr(), cu_seqlens_q.data_ptr(),
                      ws.data_ptr(), need, qt, qh, 0, 0, kb, kh, 0, 0, nb, row, code, code, k_fmt.encoding_code, S, hq, hkv, 128,
                      k_fmt.block_size, mb, cap, mq, PREFILL_CAUSAL, scale, 0)
    _lib.launch("tq_kv8_observe", dev, args + _REACH.pack(mass.data_ptr(), *ms, window, sinks, last, 0))
    return mass


_EVICT = struct.Struct("@7Q9q12i")


def evict_paged8(
    k_cache: torch.Tensor,
    k_fmt: Paged8Format,
    v_cache: torch.Tensor,
    v_fmt: Paged8Format,
    mass: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    keep: int,
    recent: int = 0,
    sinks: int = 0,
    longer_than: Optional[int] = None,
    max_seq_len: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Cut every sequence of more than longer_than tokens (default: keep) to `keep` of them, in place.

    Each KV head keeps the first `sinks`, the last `recent` and, of those between, the keep - sinks - recent tokens of
    largest mass (ties: the earlier one; NaN and tokens of bad block-table entries last).  They move, in their order, to
    positions 0 .. keep - 1 of the sequence's blocks, their mass with them; rows behind them and the mass there stay as they
    were.  A block whose rows came from others takes the largest of those blocks' scales, and codes of smaller ones are
    rounded to it (to nearest even; e4m3 codes that stay normal lose nothing).  Returns int32 [S]: keep - seq_lens,
    or 0 for a sequence left as it is, the new_lens of the plan_step that gives the blocks back; seq_lens and block_tables are
    not changed.  max_seq_len: host-side bound of seq_lens (default: the tables' capacity; tokens behind it do not
    count).  Blocks must belong to one sequence; out is memory of its own.  workspace: uint8 of tq_kv8_evict_workspace_bytes(...).
    """
    dev = _lib.require_gpu("evict_paged8", k_cache, v_cache, mass, block_tables, seq_lens, out, workspace)
    nb, heads, kb, kh, vb, vh = _check_pair(k_cache, k_fmt, v_cache, v_fmt, "evict_paged8")
    if not nb or not heads:
        raise ValueError("the caches hold no blocks")
    ms = _check_mass(mass, nb, heads, k_fmt.block_size)
    S, mb, row = _check_tables(block_tables, seq_lens)
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    longer_than = keep if longer_than is None else int(longer_than)
    if keep < 1 or recent < 0 or sinks < 0 or sinks + recent > keep:
        raise ValueError(f"keep must be positive and hold sinks and recent, got keep {keep}, recent {recent}, sinks {sinks}")
    if longer_than < keep:
        raise ValueError(f"longer_than must be at least keep, got {longer_than} and {keep}")
    if out is None:
        out = torch.empty(S, dtype=torch.int32, device=dev)
    elif out.shape != (S,) or out.dtype != torch.int32 or not out.is_contiguous():
        raise ValueError("out must be int32 [num_seqs], contiguous")
    if not S:
        return out
    seq_lens = seq_lens.contiguous()
    if out.data_ptr() < seq_lens.data_ptr() + 4 * S and seq_lens.data_ptr() < out.data_ptr() + 4 * S:
        raise ValueError("out and seq_lens share memory")  # (a sequence's heads read its length while its change is written)
    cap = _bound(max_seq_len, mb, k_fmt.block_size)
    keep, longer_than = min(keep, 0x7fff0000), min(longer_than, 0x7fff0000)  # (a sequence holds no more)
    need = 0 if cap <= longer_than else _lib.lib().tq_kv8_evict_workspace_bytes(S, heads, keep, k_fmt.block_size)
    ws = _workspace(workspace, need, dev)
    args = _EVICT.pack(k_cache.data_ptr(), v_cache.data_ptr(), mass.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
                       out.data_ptr(), ws.data_ptr(), need, kb, kh, vb, vh, *ms, nb, row, k_fmt.encoding_code, S, heads, 128,
                       k_fmt.block_size, mb, cap, keep, min(recent, keep), min(sinks, keep), longer_than, 0)
    _lib.launch("tq_kv8_evict", dev, args)
    return out
