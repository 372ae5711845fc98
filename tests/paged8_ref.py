"""Plain implementations of the 8-bit cache and its attention, from the definitions, on the CPU in 64 bits."""

import math

import numpy as np
import torch

TOP = {"e4m3": 448.0, "int8": 127.0}


def exponent(top, code):
    """The smallest e >= -126 with top <= TOP 2^e."""
    if not top > 0:
        return -126
    e = math.ceil(math.log2(top / TOP[code]))
    while TOP[code] * 2.0 ** (e - 1) >= top:
        e -= 1
    while TOP[code] * 2.0 ** e < top:
        e += 1
    return max(e, -126)


def codes(y, code):
    """Scaled 64-bit values -> the values of their codes (nearest, ties to even; NaN: NaN or 0)."""
    y = np.asarray(y, dtype=np.float64)
    if code == "int8":
        return np.clip(np.rint(np.where(np.isnan(y), 0.0, y)), -127, 127)
    a = np.clip(np.abs(y), 2.0 ** -6, 448.0)
    step = 2.0 ** (np.floor(np.log2(np.where(np.isnan(a), 1.0, a))) - 3)
    with np.errstate(invalid="ignore"):
        return np.clip(np.rint(np.clip(y, -448, 448) / step) * step, -448, 448)


class Cache:
    """One cache: values of codes [blocks, heads, block, 128] and exponents [blocks, heads] (None: never written)."""

    def __init__(self, blocks, heads, block, code):
        self.val = np.zeros((blocks, heads, block, 128))
        self.exp = np.full((blocks, heads), -999, dtype=np.int64)
        self.block, self.code = block, code

    def write(self, x, slots):
        """x [T, heads, 128] (float64), slots [T]: all tokens of one call."""
        by = {}
        for t, s in enumerate(slots):
            if 0 <= s < self.val.shape[0] * self.block:
                by.setdefault(int(s) // self.block, []).append((t, int(s) % self.block))
        for b, rows in by.items():
            fresh = any(r == 0 for _, r in rows)
            for h in range(self.val.shape[1]):
                new = np.abs(np.stack([x[t, h] for t, _ in rows]))
                new = new[np.isfinite(new)]
                e = exponent(float(new.max()) if new.size else 0.0, self.code)
                old = self.exp[b, h]
                if not fresh and old > -999:
                    if e > old:
                        self.val[b, h] = codes(self.val[b, h] * 2.0 ** (int(old) - e), self.code)
                    e = max(e, int(old))
                self.exp[b, h] = e
                for t, r in rows:
                    self.val[b, h, r] = codes(x[t, h] * 2.0 ** -e, self.code)

    def values(self):
        """[blocks, heads, block, 128]; blocks that were never written hold 0."""
        e = np.where(self.exp > -999, self.exp, 0).astype(np.float64)
        return self.val * np.where(self.exp > -999, 2.0 ** e, 0.0)[..., None, None]


def pack(values, scale, fmt):
    """Tiles (uint8 [N, H, tile_bytes]) of code values [N, H, block, 128] and scales [N, H]."""
    t = torch.as_tensor(values)
    b = (t.to(torch.float32).to(torch.float8_e4m3fn) if fmt.encoding == "e4m3" else t.to(torch.int8)).view(torch.uint8)
    if fmt.layout == "values":
        b = b.reshape(*b.shape[:2], -1, 4, 128).transpose(-1, -2)
    out = torch.zeros(*t.shape[:2], fmt.tile_bytes, dtype=torch.uint8)
    out[..., :fmt.code_bytes] = b.reshape(*t.shape[:2], -1)
    out[..., fmt.code_bytes:fmt.code_bytes + 4] = torch.as_tensor(scale).to(torch.float32).reshape(*t.shape[:2], 1).view(torch.uint8)
    return out


def gather(values, table, length):
    """Rows [length, heads, 128] of a sequence and which of them are there (bad table entries are not)."""
    n, h, block, _ = values.shape
    rows, ok = np.zeros((length, h, 128)), np.zeros(length, dtype=bool)
    for t in range(length):
        b = int(table[t // block])
        if 0 <= b < n:
            rows[t], ok[t] = values[b, :, t % block], True
    return rows, ok


def attention(q, k, v, seen, sm):
    """q [rows, 128], k and v [tokens, 128], seen [rows, tokens]: softmax(sm q k) v; rows that see nothing are 0."""
    s = sm * (q @ k.T)
    s = np.where(seen, s, -np.inf)
    m = s.max(axis=1, keepdims=True) if k.shape[0] else np.zeros((q.shape[0], 1))
    with np.errstate(invalid="ignore"):
        p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0.0)), 0.0)
    l = p.sum(axis=1, keepdims=True)
    return np.where(l > 0, (p @ v) / np.where(l > 0, l, 1.0), 0.0)


def sequences(q, starts, lens, kval, vval, tables, sm, causal, capacity):
    """out [T, heads, 128] of every query row that belongs to a sequence (NaN elsewhere)."""
    q = np.asarray(q, dtype=np.float64)
    hq, hkv = q.shape[1], kval.shape[1]
    out = np.full(q.shape, np.nan)
    for s, L in enumerate(lens):
        a, b = int(starts[s]), int(starts[s + 1])
        L = max(0, min(int(L), capacity))
        k, ok = gather(kval, tables[s], L)
        v, _ = gather(vval, tables[s], L)
        n = b - a
        last = np.arange(n) + L - n if causal else np.full(n, L - 1)
        seen = (np.arange(L)[None] <= last[:, None]) & ok[None]
        for h in range(hq):
            kh = h // (hq // hkv)
            out[a:b, h] = attention(q[a:b, h], k[:, kh], v[:, kh], seen, sm)
    return out
