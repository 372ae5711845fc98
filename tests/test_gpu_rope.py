"""GPU tests of apply_rope against rotary positions in 64 bits.

Bound per element: cosine and sine are fp32 functions of an angle that fp32 holds to 2^-25 of a turn, off by at most
2 pi 2^-25 + 2^-22 < 2^-21 each; two products and a sum add 2 * 2^-24 each; with |x|, |y| the pair:
(|x| + |y|) * magnitude * (2^-21 + 2^-22), and the output's own rounding.
"""

import numpy as np
import pytest
import torch

from turboquant.core.rope import rope_turns
from turboquant.kernels.rotation import apply_rope

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotated(x, pos, turns, style, mag):
    """(result, bound) in 64 bits."""
    x = x.double().cpu().numpy()
    # (64 bits of mantissa: a 64-bit product of a position of 2^40 would be off by 2^-53 2^40 / 2 pi turns itself)
    t = np.asarray(pos, dtype=np.longdouble)[:, None] * turns.cpu().numpy().astype(np.longdouble)
    ang = 2 * np.pi * (t - np.rint(t)).astype(np.float64)
    c, s = np.cos(ang)[:, None] * mag, np.sin(ang)[:, None] * mag
    h = turns.shape[0]
    i = np.arange(h)
    a, b = (i, i + h) if style == "half" else (2 * i, 2 * i + 1)
    out, lim = x.copy(), np.zeros_like(x)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    lim[..., a] = lim[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * mag * (2.0 ** -21 + 2.0 ** -22)
    return out, lim


def check(got, x, pos, turns, style, mag=1.0):
    want, lim = rotated(x, pos, turns, style, mag)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= lim + HALF[got.dtype] * np.abs(want)), np.max(err)
    assert torch.equal(got[..., 2 * turns.shape[0]:], x[..., 2 * turns.shape[0]:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [2, 10, 16, 48, 64, 126, 128])
@pytest.mark.parametrize("T,hq,hk", [(1, 32, 8), (3, 5, 1), (130, 8, 2), (3000, 2, 1)])
def test_apply_rope(dev, dtype, style, rot, T, hq, hk):
    g = torch.Generator().manual_seed(rot + T)
    q, k = (torch.randn(T, h, 128, generator=g).to(dtype).to(dev) for h in (hq, hk))
    pos = torch.randint(0, 200000, (T,), generator=g, dtype=torch.int32)
    turns, mag = rope_turns(rot, theta=1e6, scaling="by_parts", factor=4.0, trained_length=4096, device=dev)
    q2, k2 = apply_rope(q, k, pos.to(dev), turns, style=style, magnitude=mag)
    check(q2, q, pos.numpy(), turns, style, mag)
    check(k2, k, pos.numpy(), turns, style, mag)
    qi, ki = q.clone(), k.clone()
    r = apply_rope(qi, ki, pos.to(dev), turns, style=style, magnitude=mag, q_out=qi, k_out=ki)
    assert r[0] is qi and r[1] is ki and torch.equal(qi, q2) and torch.equal(ki, k2)


def test_apply_rope_positions(dev):
    """Far, negative and 64-bit positions; a turn back undoes a turn; k left out; no tokens."""
    turns, _ = rope_turns(128, device=dev)
    q = torch.randn(7, 4, 128, device=dev)
    for pos in ([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789, 7], [2 ** 40, -2 ** 40 + 3, 0, 10 ** 12, 5, 6, 2 ** 33 + 1]):
        dt = torch.int32 if max(pos) < 2 ** 31 else torch.int64
        p = torch.tensor(pos, dtype=dt, device=dev)
        got, none = apply_rope(q, None, p, turns)
        assert none is None
        check(got, q, pos, turns, "half")
    p = torch.tensor([3, 14, 159, 2653, 58979, 323846, 26433], device=dev)
    there, _ = apply_rope(q, None, p, turns, style="interleaved")
    back, _ = apply_rope(there, None, -p, turns, style="interleaved")
    assert torch.allclose(back, q, atol=2.0 ** -18)
    e = apply_rope(q[:0], q[:0], p[:0], turns)
    assert e[0].shape == (0, 4, 128)


def test_apply_rope_strides(dev):
    """Slices of a fused projection in place, rows off alignment, transposed inputs, strided destinations."""
    turns, _ = rope_turns(64, device=dev)
    pos = torch.arange(50, device=dev, dtype=torch.int32)
    qkv = torch.randn(50, 12, 128, device=dev).to(torch.bfloat16)
    keep = qkv.clone()
    q, k = qkv[:, :8], qkv[:, 8:10]
    apply_rope(q, k, pos, turns, q_out=q, k_out=k)
    check(qkv[:, :8], keep[:, :8], pos.cpu().numpy(), turns, "half")
    check(qkv[:, 8:10], keep[:, 8:10], pos.cpu().numpy(), turns, "half")
    assert torch.equal(qkv[:, 10:], keep[:, 10:])
    odd = torch.randn(50 * 4 * 128 + 1, device=dev).to(torch.float16)[1:].view(50, 4, 128)
    tr = torch.randn(50, 128, 4, device=dev).to(torch.float16).transpose(1, 2)
    dst = torch.zeros(50, 128, 4, device=dev, dtype=torch.float16).transpose(1, 2)
    a, b = apply_rope(odd, tr, pos, turns, style="interleaved", k_out=dst)
    check(a, odd, pos.cpu().numpy(), turns, "interleaved")
    check(b, tr, pos.cpu().numpy(), turns, "interleaved")
    assert b is dst


def test_apply_rope_refusals(dev):
    turns, _ = rope_turns(128, device=dev)
    q = torch.zeros(3, 4, 128, device=dev)
    pos = torch.zeros(3, dtype=torch.int32, device=dev)
    for args, kw in (((q[0], None, pos, turns), {}), ((q, q[:2], pos, turns), {}), ((q, None, pos[:2], turns), {}),
                     ((q, None, pos, turns.float()), {}), ((q, None, pos, torch.zeros(65, dtype=torch.float64, device=dev)), {}),
                     ((q, None, pos, turns), dict(style="other")), ((q, None, pos, turns), dict(q_out=q[:2])),
                     ((q, None, pos, turns), dict(q_out=q.half())), ((q, None, pos, turns), dict(k_out=q)),
                     ((q.cpu(), None, pos, turns), {}), ((q[..., :64], None, pos, turns), {})):
        with pytest.raises(ValueError):
            apply_rope(*args, **kw)
    for args in ((q, q.half(), pos, turns), (q, None, pos.float(), turns), (q.double(), None, pos, turns)):
        with pytest.raises(TypeError):
            apply_rope(*args)
