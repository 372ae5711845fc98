"""Plain implementations of windows with sinks, accumulated weights and eviction, from the definitions, on the CPU in 64 bits."""

import numpy as np
import torch

import paged8_ref as ref


def visible(position, tokens, window, sinks):
    """Which of `tokens` tokens the query at `position` sees."""
    t = np.arange(tokens)
    see = t <= position
    return see if window is None else see & ((t > position - window) | (t < sinks))


def weights(q, k, see, sm):
    """Softmax weights of one query row over the tokens that it sees; none: zeros."""
    if not see.any():
        return np.zeros(k.shape[0])
    s = np.where(see, sm * (k @ q), -np.inf)
    p = np.where(see, np.exp(s - s.max()), 0.0)
    return p / p.sum()


def sequence(q, kval, vval, table, L, window, sinks, sm, last=None):
    """(out [n, hq, 128], weights [hkv, L]) of the last n tokens' queries; the weights' sum runs over the last `last` of them."""
    n, hq, _ = q.shape
    hkv = kval.shape[1]
    k, ok = ref.gather(kval, table, L)
    v = ref.gather(vval, table, L)[0] if vval is not None else None
    out, mass = np.zeros((n, hq, 128)), np.zeros((hkv, L))
    for i in range(n):
        see = visible(L - n + i, L, window, sinks) & ok
        for h in range(hq):
            w = weights(q[i, h], k[:, h // (hq // hkv)], see, sm)
            if v is not None:
                out[i, h] = w @ v[:, h // (hq // hkv)]
            if last is None or i >= n - last:
                mass[h // (hq // hkv)] += w
    return out, mass


def accumulate(mass, add, table, L, new, block):
    """mass [blocks, heads, block] after a call that gave `add` [heads, L]; in place."""
    for t in range(L):
        b = int(table[t // block])
        if 0 <= b < mass.shape[0]:
            mass[b, :, t % block] = (0.0 if t >= L - new else mass[b, :, t % block]) + add[:, t]


def order(mass):
    """Numbers by which the heaviest come first: NaN below all."""
    return np.where(np.isnan(mass), -np.inf, mass), np.isnan(mass)


def chosen(mass, ok, L, keep, recent, sinks):
    """The kept tokens of a sequence of one KV head, in order: mass [L], ok [L] (a good table entry)."""
    body = list(range(sinks, L - recent))
    # the worst: bad entries and NaN, one as the other; then by size
    rank = sorted(body, key=lambda t: (0 if not ok[t] or np.isnan(mass[t]) else -1, 0.0 if not ok[t] or np.isnan(mass[t]) else -mass[t], t))
    return sorted(list(range(sinks)) + rank[:keep - sinks - recent] + list(range(L - recent, L)))


def evict(val, exp, mass, tables, lens, keep, recent, sinks, longer_than, cap, block, code):
    """In place: val two arrays of code values [blocks, heads, block, 128], exp two of exponents [blocks, heads] (-999: scale 0),
    mass [blocks, heads, block].  Returns the changes."""
    change = []
    for table, length in zip(tables, lens):
        L = max(0, min(int(length), cap))
        if L <= longer_than:
            change.append(0)
            continue
        change.append(keep - int(length))
        nb = mass.shape[0]
        blk = np.array([int(table[t // block]) for t in range(L)])
        ok = (blk >= 0) & (blk < nb)
        src_val, src_exp, src_mass = [v.copy() for v in val], [e.copy() for e in exp], mass.copy()
        for h in range(mass.shape[1]):
            m = np.array([src_mass[blk[t], h, t % block] if ok[t] else np.nan for t in range(L)])
            src = chosen(m, ok, L, keep, recent, sinks)
            for b0 in range(0, keep, block):
                rows = range(b0, min(b0 + block, keep))
                to = blk[b0]
                for i in range(2):
                    es = [src_exp[i][blk[src[d]], h] if ok[src[d]] else -999 for d in rows]
                    top = max(es)
                    if not 0 <= to < nb:
                        continue
                    exp[i][to, h] = top
                    for d, e in zip(rows, es):
                        t = src[d]
                        x = src_val[i][blk[t], h, t % block] if ok[t] else np.zeros(128)
                        val[i][to, h, d - b0] = x if e == top and e > -999 else ref.codes(x * (2.0 ** (e - top) if e > -999 else 0.0), code)
                if 0 <= to < nb:
                    for d in rows:
                        t = src[d]
                        mass[to, h, d - b0] = src_mass[blk[t], h, t % block] if ok[t] else 0.0
    return change


def read(cache, fmt):
    """(code values, exponents) of a cache's tiles; scale 0: -999."""
    n = fmt.code_bytes
    c = cache.cpu()
    b = c[..., :n].contiguous()
    if fmt.layout == "values":
        b = b.view(*b.shape[:2], -1, 128, 4).transpose(-1, -2).contiguous()
    dt = torch.float8_e4m3fn if fmt.encoding == "e4m3" else torch.int8
    val = b.view(*b.shape[:2], fmt.block_size, 128).view(dt).to(torch.float64).numpy().copy()
    scale = c[..., n:n + 4].contiguous().view(torch.float32)[..., 0].double().numpy()
    return val, np.where(scale > 0, np.log2(np.where(scale > 0, scale, 1.0)), -999).astype(np.int64)
