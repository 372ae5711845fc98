"""Paged K/V cache of 8 bits a value: format, quantisation into slots, decode and prefill attention.

For the layers that the packed 2..4-bit formats are too coarse for (the boundary layers of
integration.paged_backend, protected_bits=8).  One tensor per K or V cache, uint8 [num_blocks,
num_kv_heads, tile_bytes]; the tile of (physical block, KV head) holds

    [block_size x 128 codes][fp32 scale][12 unused bytes]

and a code stands for code * scale.  Codes are e4m3 ("e4m3") or two's complement ("int8"), the scale is the
smallest power of two that takes the tile's largest finite value, so a change of scale moves exponents
only.  Keys are row-major [block_size][128]; values interleave the dims of four consecutive tokens, byte
512 g + 4 d + r = dim d of token 4 g + r, the 8-bit case of the "values" layout of kernels.paged.

Slot addressing, block tables and lengths are those of kernels.paged; there is no rotation here (scores do not
change when q and k are rotated alike, and values come back in the basis they were stored in).
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from typing import Optional

import torch

from turboquant import _lib
from turboquant.kernels.paged import PREFILL_CAUSAL, allocate_cache  # noqa: F401  (allocate_cache: any tile format)

_ENCODINGS = {"e4m3": 0, "int8": 1}
_CODE_DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SCALE_BYTES = 16


@dataclass(frozen=True)
class Paged8Format:
    """Geometry of one 8-bit paged cache.  layout: "keys" for a K cache, "values" for a V cache.

    code_bytes and tile_bytes: bytes of a tile's codes and of the whole tile."""

    encoding: str = "e4m3"
    block_size: int = 16
    layout: str = "keys"
    head_dim: int = 128

    def __post_init__(self):
        if self.encoding not in _ENCODINGS:
            raise ValueError(f"encoding must be one of {sorted(_ENCODINGS)}, got {self.encoding!r}")
        if self.block_size <= 0 or self.block_size % 16 or self.block_size > 65536:
            raise ValueError(f"block_size must be a multiple of 16 in 16..65536, got {self.block_size}")
        if self.layout not in ("keys", "values"):
            raise ValueError(f"layout must be 'keys' or 'values', got {self.layout!r}")
        if self.head_dim != 128:
            raise ValueError("head_dim must be 128")
        # (worked out once: every call reads them)
        object.__setattr__(self, "code_bytes", self.block_size * self.head_dim)
        object.__setattr__(self, "tile_bytes", self.code_bytes + SCALE_BYTES)
        object.__setattr__(self, "encoding_code", _ENCODINGS[self.encoding])

    @classmethod
    def for_keys(cls, encoding: str = "e4m3", block_size: int = 16) -> "Paged8Format":
        return cls(encoding, block_size, "keys")

    @classmethod
    def for_values(cls, encoding: str = "e4m3", block_size: int = 16) -> "Paged8Format":
        return cls(encoding, block_size, "values")


def dequantize_paged8(cache: torch.Tensor, fmt: Paged8Format) -> torch.Tensor:
    """The values a cache holds: fp32 [num_blocks, num_kv_heads, block_size, 128] (torch operations, any device)."""
    _check_cache(cache, fmt, "dequantize_paged8")
    n = fmt.code_bytes
    codes = cache[..., :n].contiguous()
    if fmt.layout == "values":
        codes = codes.view(*codes.shape[:2], -1, 128, 4).transpose(-1, -2).contiguous()
    x = codes.view(*codes.shape[:2], fmt.block_size, 128).view(_CODE_DTYPE[fmt.encoding]).to(torch.float32)
    return x * cache[..., n:n + 4].contiguous().view(torch.float32)[..., None]


def _check_cache(cache: torch.Tensor, fmt: Paged8Format, what: str) -> tuple[int, int]:
    """The cache's block and head strides."""
    if cache.dtype != torch.uint8 or cache.dim() != 3:
        raise ValueError(f"{what}: cache must be uint8 [num_blocks, num_kv_heads, tile_bytes]")
    sb, sh, s1 = cache.stride()
    if cache.shape[2] < fmt.tile_bytes or s1 != 1:
        raise ValueError(f"{what}: cache tiles must hold {fmt.tile_bytes} contiguous bytes")
    if (sb | sh | cache.data_ptr()) % 16:
        raise ValueError(f"{what}: cache tiles must be 16-byte aligned")
    return sb, sh


def _check_pair(k_cache, k_fmt, v_cache, v_fmt, what: str) -> tuple[int, int, int, int, int, int]:
    """(blocks, heads, K block stride, K head stride, V block stride, V head stride)."""
    kb, kh = _check_cache(k_cache, k_fmt, what)
    vb, vh = _check_cache(v_cache, v_fmt, what)
    if k_fmt.layout != "keys" or v_fmt.layout != "values":
        raise ValueError(f"{what}: the K cache takes layout='keys', the V cache layout='values'")
    if k_fmt.block_size != v_fmt.block_size or k_fmt.encoding != v_fmt.encoding:
        raise ValueError(f"{what}: K and V caches must share block_size and encoding")
    nb, heads, _ = k_cache.shape
    if v_cache.shape[0] != nb or v_cache.shape[1] != heads:
        raise ValueError(f"{what}: K and V caches must have the same [num_blocks, num_kv_heads]")
    return nb, heads, kb, kh, vb, vh


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [T, H, 128] with rows that the kernels can load: itself, or a contiguous copy."""
    st, sh, s1 = x.stride()
    return x if s1 == 1 and not (st | sh) % 8 and not x.data_ptr() % 16 else x.clone(memory_format=torch.contiguous_format)


_UPDATE = struct.Struct("@2Q4q2Q4qQ2q6i")


def quantize_paged8_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_fmt: Paged8Format,
    v_fmt: Paged8Format,
):
    """Quantise k and v [T, Hkv, 128] (f32/f16/bf16) into their slots of the paged caches, one launch.

    Negative slots, and slots behind the cache, are skipped.  A block that is written from its first row on
    starts anew: its scale is that of the new rows alone and its other rows hold nothing.
    Otherwise a block's scale only grows, and its other rows are requantised when it does.  The tokens of one
    call that go to one block must follow each other with consecutive slots, as a sequence's new tokens do (up
    to 63 skipped tokens between two of them); a block for which that does not hold, or a slot named
    twice, has unspecified contents afterwards.
    """
    dev = _lib.require_gpu("quantize_paged8_kv", k, v, slot_mapping, k_cache, v_cache)
    if k.dim() != 3 or k.shape[2] != 128 or v.shape != k.shape:
        raise ValueError(f"k and v must both be [T, H, 128], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != v.dtype:
        raise TypeError("k and v must share a dtype")
    T, H, _ = k.shape
    nb, heads, kb, kc, vb, vc = _check_pair(k_cache, k_fmt, v_cache, v_fmt, "quantize_paged8_kv")
    if heads != H:
        raise ValueError(f"caches have {heads} heads, k and v {H}")
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != T:
        raise ValueError("slot_mapping must be [T]")
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise TypeError("slot_mapping must be int32 or int64")
    k, v, slot_mapping = _rows(k), _rows(v), slot_mapping.contiguous()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    args = _UPDATE.pack(k.data_ptr(), v.data_ptr(), kt, kh, vt, vh, k_cache.data_ptr(), v_cache.data_ptr(), kb, kc, vb, vc,
                        slot_mapping.data_ptr(), T, nb, _lib.dtype_code(k), _lib.dtype_code(slot_mapping),
                        k_fmt.encoding_code, H, 128, k_fmt.block_size)
    _lib.launch("tq_kv8_update", dev, args)
    return k_cache, v_cache


_ATTN = struct.Struct("@8Q11q12ifi")
_SCALE = 1.0 / math.sqrt(128)


def _attention(name, dev, q, caches, k_cache, v_cache, k_fmt, block_tables, seq_lens, cu_seqlens_q, sm_scale, max_seq_len,
               max_q_len, flags, out, workspace):
    rows, hq, _ = q.shape
    nb, hkv, kb, kh, vb, vh = caches
    S, mb = block_tables.shape if block_tables.dim() == 2 else (-1, 0)
    if S != seq_lens.shape[0] or (mb > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [num_seqs, max_blocks] with unit inner stride")
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    if not hkv or hq % hkv:
        raise ValueError(f"num_q_heads {hq} must be a multiple of num_kv_heads {hkv}")
    if not nb:
        raise ValueError("the caches hold no blocks")
    if out is not None and (out.shape != q.shape or out.device != q.device):
        raise ValueError("out must have q's shape and device")
    scale = _SCALE if sm_scale is None else float(sm_scale)
    if not math.isfinite(scale):
        raise ValueError("sm_scale must be finite")
    seq_lens = seq_lens.contiguous()
    q = _rows(q)
    if out is None:
        out = torch.empty_like(q)
    if not rows or not hq:
        return out
    target = out
    ot, oh, o1 = out.stride()
    if (rows > 1 and not ot) or (hq > 1 and not oh):
        raise ValueError("rows of out share memory")
    if o1 != 1 or (ot | oh) % 8 or out.data_ptr() % 16:
        # a destination that takes no vector stores gets a copy of the result (rows of no sequence stay as they were)
        target = out.clone(memory_format=torch.contiguous_format)
        ot, oh, _ = target.stride()
    L = _lib.lib()
    if cu_seqlens_q is None:
        need = L.tq_kv8_decode_workspace_bytes(S, hq, hkv)
    else:
        need = L.tq_kv8_prefill_workspace_bytes(S, max_q_len, hq, hkv, mb, k_fmt.block_size)
    if workspace is None:
        # (a buffer of this call: of the current stream, and of the graph under capture)
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.get_device() != dev.index or workspace.numel() * workspace.element_size() < need or \
            workspace.data_ptr() % 256 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be {need} contiguous bytes on {dev}, 256-byte aligned")
    qt, qh, _ = q.stride()
    args = _ATTN.pack(q.data_ptr(), target.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
                      seq_lens.data_ptr(), 0 if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), workspace.data_ptr(), need,
                      qt, qh, ot, oh, kb, kh, vb, vh, nb, block_tables.stride(0) if S > 1 else mb, _lib.dtype_code(q),
                      _lib.dtype_code(target), k_fmt.encoding_code, S, hq, hkv, 128, k_fmt.block_size, mb, max_seq_len,
                      max_q_len, flags, scale, 0)
    _lib.launch(name, dev, args)
    if target is not out:
        out.copy_(target)
    return out


def decode_paged8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    k_fmt: Paged8Format,
    v_cache: torch.Tensor,
    v_fmt: Paged8Format,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    max_seq_len: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of one query token per sequence, q [S, Hq, 128], over 8-bit paged K/V caches.

    block_tables int32 [S, max_blocks] (entries outside the cache mask their tokens), seq_lens int32 [S];
    max_seq_len: host-side bound of seq_lens (default: the tables' capacity; longer sequences are cut there).
    Up to 16 query heads per KV head.  Output dtype = out.dtype or q.dtype; a row's q and probabilities are rounded
    to fp16 (probabilities below 2^-39 of the row's largest count as zero), with f32 on either side they are
    carried in twice the precision.  V enters relative to the largest scale so far of the sequence's blocks: exact
    down to 2^-15 of it, zero below 2^-24.  A sequence of length 0 gives zeros; a NaN in the cache reaches the
    heads that see it.  workspace: uint8 of tq_kv8_decode_workspace_bytes(...) for callers that keep one (calls that
    overlap must not share it).
    """
    dev = _lib.require_gpu("decode_paged8", q, k_cache, v_cache, block_tables, seq_lens, out, workspace)
    if q.dim() != 3 or q.shape[2] != 128:
        raise ValueError("q must be [S, Hq, 128]")
    if seq_lens.dim() != 1 or seq_lens.shape[0] != q.shape[0]:
        raise ValueError("seq_lens must be [S]")
    caches = _check_pair(k_cache, k_fmt, v_cache, v_fmt, "decode_paged8")
    if caches[1] and q.shape[1] > 16 * caches[1]:
        raise ValueError("decode_paged8 takes up to 16 query heads per KV head")
    cap = min(block_tables.shape[-1] * k_fmt.block_size, 0x7fff0000) if block_tables.dim() else 0
    msl = cap if max_seq_len is None else max(0, min(int(max_seq_len), cap))
    return _attention("tq_kv8_decode", dev, q, caches, k_cache, v_cache, k_fmt, block_tables, seq_lens, None, sm_scale, msl, 1,
                      0, out, workspace)


def prefill_paged8(
    q: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    k_cache: torch.Tensor,
    k_fmt: Paged8Format,
    v_cache: torch.Tensor,
    v_fmt: Paged8Format,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    causal: bool = True,
    max_q_len: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of several new tokens per sequence, q [T, Hq, 128], over 8-bit paged K/V caches.

    Sequence s owns query rows cu_seqlens_q[s] .. cu_seqlens_q[s+1] - 1 (int32 [S+1], device, ascending, at most T) and
    seq_lens[s] cache tokens, the new ones included.  causal: query i of n sees the tokens up to position
    seq_lens - n + i, otherwise all of them; a row that sees none gives zeros, and NaN in the cache reaches
    the rows that see it alone.  Any number of query heads per KV head.
    max_q_len: host-side bound of the query counts (default: T).  Rows of q that belong to no sequence are
    left as they were in out.  Types, roundings and workspace as in decode_paged8, but 16-bit calls round probabilities below
    2^-18 of the row's largest to fewer bits and those below 2^-29 to zero.
    """
    dev = _lib.require_gpu("prefill_paged8", q, cu_seqlens_q, k_cache, v_cache, block_tables, seq_lens, out, workspace)
    if q.dim() != 3 or q.shape[2] != 128:
        raise ValueError("q must be [T, Hq, 128]")
    if seq_lens.dim() != 1 or cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] != seq_lens.shape[0] + 1:
        raise ValueError("seq_lens must be [num_seqs] and cu_seqlens_q [num_seqs + 1]")
    if cu_seqlens_q.dtype != torch.int32:
        raise TypeError("cu_seqlens_q must be int32")
    caches = _check_pair(k_cache, k_fmt, v_cache, v_fmt, "prefill_paged8")
    T = q.shape[0]
    mq = T if max_q_len is None else max(0, min(int(max_q_len), T))
    return _attention("tq_kv8_prefill", dev, q, caches, k_cache, v_cache, k_fmt, block_tables, seq_lens,
                      cu_seqlens_q.contiguous(), sm_scale, 0, mq, PREFILL_CAUSAL if causal else 0, out, workspace)
