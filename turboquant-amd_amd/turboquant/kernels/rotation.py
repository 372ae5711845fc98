"""Stand-alone rotations of 128-element query / key rows on the GPU: Walsh-Hadamard and rotary positions.

wht_rows(x) = x @ make_wht_matrix(128) (the matrix is symmetric and its own inverse), computed
with fp32 butterflies by tq_wht_rows.  It is the operation of the reference backend's
TurboQuantFP8State.rotate_query / rotate_output (integration/vllm_backend.py:158-177) for
callers that rotate outside the decode call; decode_paged(..., rotate=True) fuses both
rotations into the decode kernels instead.

apply_rope turns the pairs of every row by its token's position (the step before the cache write and, for
queries, before attention); the frequencies come from turboquant.core.rope.
"""

from __future__ import annotations

import struct
from typing import Optional

import torch

from turboquant import _lib


def wht_rows(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ make_wht_matrix(128) over the last dimension (f32 / f16 / bf16 GPU tensors).

    out: optional destination of x's shape (any of the three dtypes); it may be x itself.
    """
    _lib.require_gpu("wht_rows", x)
    if x.dim() < 1 or x.shape[-1] != 128:
        raise ValueError("the last dimension must be 128")
    if out is None:
        out = torch.empty_like(x)
    if out.shape != x.shape or out.device != x.device:
        raise ValueError("out must have x's shape and device")

    def rows3(t: torch.Tensor) -> torch.Tensor:
        if t.dim() == 3 and t.stride(2) == 1:
            return t
        if t.dim() == 2 and t.stride(1) == 1:
            return t.unsqueeze(1)
        return t.reshape(-1, 1, 128) if t.is_contiguous() else None

    xs = rows3(x)
    if xs is None:
        xs = rows3(x.contiguous())
    os_ = rows3(out)
    target = out
    if os_ is None:  # a non-contiguous destination of another shape: write a copy back
        target = torch.empty_like(x, memory_format=torch.contiguous_format)
        os_ = rows3(target)
    if xs.shape[0] * xs.shape[1] == 0:
        return out
    rc = _lib.lib().tq_wht_rows(
        xs.data_ptr(), _lib.dtype_code(xs), xs.stride(0), xs.stride(1), xs.shape[0], xs.shape[1], 128,
        os_.data_ptr(), _lib.dtype_code(os_), os_.stride(0), os_.stride(1), _lib.stream_handle(x.device))
    _lib.check(rc, "tq_wht_rows")
    if target is not out:
        out.copy_(target)
    return out


_ROPE = struct.Struct("@4Q8q2Qq7if")
_STYLES = {"half": 0, "interleaved": 1}


def _rope_pair(x: torch.Tensor, out: Optional[torch.Tensor]):
    """(source, what the kernel writes, the destination, their token and head strides)."""
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError("destinations must have their input's shape and dtype")
    xt, xh, x1 = x.stride()
    ot, oh, o1 = out.stride()
    if (not ot and out.shape[0] > 1) or (not oh and out.shape[1] > 1):
        raise ValueError("rows of a destination share memory")
    dst = out
    if o1 != 1 or (out.data_ptr() == x.data_ptr() and (ot != xt or oh != xh)):
        dst = torch.empty_like(x, memory_format=torch.contiguous_format)
        ot, oh, _ = dst.stride()
    if x1 != 1:
        x = x.contiguous()
        xt, xh, _ = x.stride()
    return x, dst, out, (xt, xh, ot, oh)


def apply_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    turns: torch.Tensor,
    style: str = "half",
    magnitude: float = 1.0,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
):
    """Rotary positions on q [T, Hq, 128] and k [T, Hk, 128] (one dtype of f32 / f16 / bf16); k may be None.

    turns: fp64 [rotary_dim / 2] on the device, the turns of each pair per position (core.rope.rope_turns);
    positions: int32 or int64 [T], negative ones turn back.  With angle a = 2 pi * position * turns[i] pair
    i of a row goes to magnitude * (x cos a - y sin a, y cos a + x sin a); angles are reduced in 64 bits.
    style: "half" pairs element i with i + rotary_dim / 2, "interleaved" 2i with 2i + 1.  Elements from
    rotary_dim on are copied.  q_out / k_out: destinations of the same shape and dtype, which may be the
    inputs themselves.  Returns (q_out, k_out).
    """
    dev = _lib.require_gpu("apply_rope", q, k, positions, turns, q_out, k_out)
    if style not in _STYLES:
        raise ValueError(f"style must be one of {sorted(_STYLES)}, got {style!r}")
    if turns.dtype != torch.float64 or turns.dim() != 1 or not 1 <= turns.shape[0] <= 64:
        raise ValueError("turns must be float64 [rotary_dim / 2] with rotary_dim <= 128")
    if q.dim() != 3 or q.shape[2] != 128:
        raise ValueError(f"q must be [T, Hq, 128], got {tuple(q.shape)}")
    T = q.shape[0]
    if k is not None and (k.dim() != 3 or k.shape[0] != T or k.shape[2] != 128):
        raise ValueError(f"k must be [{T}, Hk, 128], got {tuple(k.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("q and k must share a dtype")
    if positions.dim() != 1 or positions.shape[0] != T:
        raise ValueError("positions must be [T]")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64")
    if k is None and k_out is not None:
        raise ValueError("k_out needs k")
    turns, positions = turns.contiguous(), positions.contiguous()

    q, qd, q_out, qs = _rope_pair(q, q_out)
    kd, kp, kdp, hk, ks = None, 0, 0, 0, (0, 0, 0, 0)
    if k is not None:
        k, kd, k_out, ks = _rope_pair(k, k_out)
        kp, kdp, hk = k.data_ptr(), kd.data_ptr(), k.shape[1]
    if T:
        args = _ROPE.pack(q.data_ptr(), kp, qd.data_ptr(), kdp, qs[0], qs[1], ks[0], ks[1], qs[2], qs[3], ks[2], ks[3],
                          positions.data_ptr(), turns.data_ptr(), T, _lib.dtype_code(q), _lib.dtype_code(positions), q.shape[1],
                          hk, 128, 2 * turns.shape[0], _STYLES[style], float(magnitude))
        _lib.launch("tq_rope", dev, args)
    if qd is not q_out:
        q_out.copy_(qd)
    if kd is not k_out:
        k_out.copy_(kd)
    return q_out, k_out
