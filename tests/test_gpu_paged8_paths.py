"""8-bit paged cache: calls of more than 64 sequences, runs with skipped tokens over several sub-tiles, NaN that decode sees."""

import math

import numpy as np
import pytest
import torch

import paged8_ref as ref
from test_gpu_paged8 import bound, formats, rows64, same_bits
from test_gpu_paged8_edges import filled
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import decode_paged8, dequantize_paged8, prefill_paged8, quantize_paged8_kv

pytestmark = pytest.mark.gpu


def lengths(kind, seqs):
    """(past, new) of each sequence; every 7th, and the 64th, has no new tokens."""
    rng = np.random.default_rng(seqs)
    if kind == "whole":      # a row block each, no long keys
        past, new = rng.integers(0, 200, seqs), rng.integers(1, 16, seqs)
    elif kind == "shares":   # a few long keys among short ones: cut over the waves
        past, new = rng.integers(0, 300, seqs), rng.integers(1, 60, seqs)
        past[[3, 64, seqs - 1]] = 9000, 7001, 5003
    else:                    # many row blocks of like lengths
        past, new = rng.integers(0, 9, seqs), rng.integers(110, 140, seqs)
    new[1::7] = 0
    new[63] = 0
    new[[64, seqs - 1]] = np.maximum(new[[64, seqs - 1]], 1)
    return past, new


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind,seqs,hkv,group", [("whole", 65, 2, 4), ("whole", 200, 1, 3), ("shares", 66, 2, 4), ("shares", 200, 1, 6),
                                                 ("tickets", 160, 8, 4), ("tickets", 200, 8, 4)])
def test_prefill_many_sequences(dev, dtype, kind, seqs, hkv, group):
    past, new = lengths(kind, seqs)
    lens = (past + new).tolist()
    starts = np.concatenate([[0], np.cumsum(new)])
    block = 16
    kf, vf = formats("e4m3", block)
    need = [-(-n // block) for n in lens]
    nb = sum(need) + 1
    g = torch.Generator(device=dev).manual_seed(seqs)
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seqs))
    bt = torch.full((seqs, max(need)), -1, dtype=torch.int32)
    slots, at = [], 0
    for s, b in enumerate(need):
        bt[s, :b] = perm[at:at + b]
        at += b
        t = torch.arange(lens[s])
        slots.append(bt[s].long()[t // block] * block + t % block)
    slots, bt = torch.cat(slots).to(dev), bt.to(dev)
    kc, vc = (allocate_cache(nb, hkv, f, device=dev) for f in (kf, vf))
    k, v = (torch.randn(slots.numel(), hkv, 128, generator=g, device=dev) for _ in range(2))
    quantize_paged8_kv(k, v, slots, kc, vc, kf, vf)
    q = torch.randn(int(starts[-1]) + 1, hkv * group, 128, generator=g, device=dev).to(dtype)
    cu, sl = (torch.tensor(np.asarray(x), dtype=torch.int32, device=dev) for x in (starts, lens))
    out = torch.full_like(q, 3.0)
    prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=int(new.max()), out=out)
    assert torch.equal(out, prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=int(new.max()), out=torch.full_like(q, 3.0)))
    assert torch.all(out[-1] == 3.0)
    kval, vval = dequantize_paged8(kc, kf).double(), dequantize_paged8(vc, vf).double()
    d = dict(kf=kf, bt=bt)
    top = float(vval.abs().max())
    for s in range(seqs):
        rows = slice(int(starts[s]), int(starts[s + 1]))
        for h in {0, hkv * group - 1} if new[s] else ():
            want = rows64(q, d, kval, vval, lens, starts, s, h, group).cpu().numpy()
            err = np.abs(out[rows, h].double().cpu().numpy() - want)
            assert np.all(err <= bound(top, lens[s], dtype, dtype, want)), (s, h)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [48, 128])
@pytest.mark.parametrize("ranks", [1, 3, 64])
@pytest.mark.parametrize("odd", [False, True])
def test_quantize_long_runs_between_others(dev, code, block, ranks, odd):
    """Every ranks-th token has a slot: runs over several 16-row sub-tiles that begin inside one, in calls that meet inside a
    block and whose rows grow, with NaN and infinities in later sub-tiles."""
    n, first = 2 * block + 9, 5
    kf, vf = formats(code, block)
    blk = [4, 0, 2]
    slots = torch.full((n * ranks,), -1, dtype=torch.int64)
    slots[ranks - 1::ranks] = torch.tensor([blk[i // block] * block + i % block for i in range(first, first + n)])
    x = [torch.randn(n * ranks, 2, 128, generator=torch.Generator().manual_seed(ranks + i)) for i in range(2)]
    cuts = [0, 21 * ranks + 1, (block + 19) * ranks, n * ranks]
    for i, c in enumerate(cuts[1:-1]):
        for y in x:
            y[c:] *= (1.5, 40.0)[i]
    if odd:
        for y in x:
            y[(block - 3) * ranks + ranks - 1, 0, 7] = float("nan")
            y[30 * ranks + ranks - 1, 1, 100] = float("inf")
            y[(block + 20) * ranks + ranks - 1, :, 3] = float("-inf")
            y[(block + 25) * ranks + ranks - 1, 1, 90] = float("nan")
    x = [y.to(torch.bfloat16) for y in x]
    caches = [allocate_cache(6, 2, f, device=dev) for f in (kf, vf)]
    want = [ref.Cache(6, 2, block, code) for _ in range(2)]
    for a, b in zip(cuts, cuts[1:]):
        quantize_paged8_kv(x[0][a:b].to(dev), x[1][a:b].to(dev), slots[a:b].to(dev), *caches, kf, vf)
        for w, y in zip(want, x):
            w.write(y[a:b].double().numpy(), slots[a:b].tolist())
    for c, w, f in zip(caches, want, (kf, vf)):
        same_bits(c, w, f)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[40, 61], [5000, 33], [64, 4000, 17]])
def test_decode_nan_of_the_cache(dev, dtype, lens):
    """A NaN in V reaches its dim of the heads that see its token, one in K all dims, for sequences that one wave takes and for
    cut ones; all other outputs keep the bits that they have with 0 in those places."""
    g = torch.Generator(device=dev).manual_seed(len(lens))
    hkv, group, block = 2, 4, 16
    sets = []
    for bad in (float("nan"), 0.0):
        g.manual_seed(len(lens))
        parts = []
        for s, n in enumerate(lens):
            k, v = (torch.randn(n, hkv, 128, generator=g, device=dev) for _ in range(2))
            v[n // 2, s % 2, 5] = bad
            v[n - 1, s % 2, 127] = bad
            if s == 1:
                k[n // 3, 1, 9] = bad
            parts.append(filled(k, v, "e4m3", block, dev)[0])
        # one pool of all sequences' blocks
        base = np.cumsum([0] + [p[0].shape[0] for p in parts])
        bt = torch.full((len(lens), max(p[4].shape[1] for p in parts)), -1, dtype=torch.int32, device=dev)
        for s, p in enumerate(parts):
            bt[s, :p[4].shape[1]] = p[4][0] + int(base[s])
        kc, vc = (torch.cat([p[i] for p in parts]) for i in (0, 2))
        q = torch.randn(len(lens), hkv * group, 128, generator=g, device=dev).to(dtype)
        sl = torch.tensor(lens, dtype=torch.int32, device=dev)
        sets.append(decode_paged8(q, kc, parts[0][1], vc, parts[0][3], bt, sl))
    want = sets[1].clone().view(len(lens), hkv, group, 128)
    for s in range(len(lens)):
        want[s, s % 2, :, [5, 127]] = float("nan")
        if s == 1:
            want[s, 1] = float("nan")
    want = want.view_as(sets[0])
    assert not bool(torch.isnan(sets[1]).any())
    assert torch.equal(torch.isnan(sets[0]), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(sets[0]), torch.nan_to_num(want))
