"""8-bit paged cache: NaN and far scales behind the causal mask, sequences of 2^31 tokens, empty tables, calls side by side,
tokens with others' in between."""

import math

import numpy as np
import pytest
import torch

import paged8_ref as ref
from test_gpu_paged8 import SM, bound, formats, same_bits
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import decode_paged8, dequantize_paged8, prefill_paged8, quantize_paged8_kv

pytestmark = pytest.mark.gpu


def filled(k, v, code, block, dev, blocks=None):
    """Caches that hold one sequence's rows k and v [L, hkv, 128] in shuffled blocks, and its table."""
    need = -(-k.shape[0] // block)
    kf, vf = formats(code, block)
    kc, vc = (allocate_cache(blocks or need + 2, k.shape[1], f, device=dev) for f in (kf, vf))
    perm = torch.randperm(kc.shape[0], generator=torch.Generator().manual_seed(need))[:need].to(dev)
    t = torch.arange(k.shape[0], device=dev)
    quantize_paged8_kv(k, v, perm[t // block] * block + t % block, kc, vc, kf, vf)
    bt = perm.to(torch.int32)[None]
    kval, vval = (dequantize_paged8(c, f)[perm].transpose(1, 2).reshape(-1, k.shape[1], 128)[:k.shape[0]].double()
                  for c, f in ((kc, kf), (vc, vf)))
    return (kc, kf, vc, vf, bt), kval, vval


def causal64(q, kval, vval, past):
    """Row by row over the tokens that it sees, all others left out."""
    group = q.shape[1] // kval.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for i in range(q.shape[0]):
        for h in range(q.shape[1]):
            n = past + i + 1
            p = torch.softmax(kval[:n, h // group] @ q[i, h].double() * SM, 0)
            out[i, h] = (p[:, None] * vval[:n, h // group]).sum(0)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("past,block,hkv", [(100, 16, 2), (0, 48, 1), (6000, 16, 1)])
def test_prefill_nan_stays_behind_the_mask(dev, dtype, past, block, hkv):
    """A token with NaN in K or V reaches the rows that see it, in its dims, and no row before it."""
    g = torch.Generator(device=dev).manual_seed(past + 1)
    new = 90
    k, v = (torch.randn(past + new, hkv, 128, generator=g, device=dev) for _ in range(2))
    v[past + 2, 0, 7] = float("nan")
    v[past + 30, 0, 3] = float("nan")
    v[past + 31] = float("nan")
    k[past + 70, hkv - 1, 5] = float("nan")
    if past:
        v[past // 2, 0, 100] = float("nan")
    args, kval, vval = filled(k, v, "e4m3", block, dev)
    q = torch.randn(new, 4 * hkv, 128, generator=g, device=dev).to(dtype)
    cu = torch.tensor([0, new], dtype=torch.int32, device=dev)
    sl = torch.tensor([past + new], dtype=torch.int32, device=dev)
    got = prefill_paged8(q, cu, *args, sl)
    want = causal64(q, kval, vval, past)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert bool(ok[0].any()) and not bool(ok[-1].any(dim=-1)[0])
    top = float(torch.nan_to_num(vval).abs().max())
    w = want[ok].cpu().numpy()
    assert np.all(np.abs(got.double()[ok].cpu().numpy() - w) <= bound(top, past + new, dtype, got.dtype, w))
    # without a mask every row sees all of them
    every = prefill_paged8(q, cu, *args, sl, causal=False)
    assert bool(torch.isnan(every).all(dim=-1).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_prefill_far_scales_behind_the_mask(dev, code, dtype):
    """Values 2^32 times larger from token 16 on: the rows before do not see them and lose nothing to them."""
    g = torch.Generator(device=dev).manual_seed(4)
    k, v = (torch.randn(64, 1, 128, generator=g, device=dev) for _ in range(2))
    v[:16] *= 2.0 ** -14
    v[16:] *= 2.0 ** 10
    v[32:48] *= 2.0 ** -30
    args, kval, vval = filled(k, v, code, 16, dev)
    q = torch.randn(64, 2, 128, generator=g, device=dev).to(dtype)
    cu, sl = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 64], [64]))
    got = prefill_paged8(q, cu, *args, sl, out=torch.empty(64, 2, 128, device=dev)).double().cpu().numpy()
    want = causal64(q, kval, vval, 0).cpu().numpy()
    for rows in (slice(0, 16), slice(16, 64)):
        top = float(vval[rows].abs().max())
        assert np.all(np.abs(got[rows] - want[rows]) <= bound(top, 64, dtype, torch.float32, want[rows]))


def test_sequences_of_2_31_tokens(dev):
    """A table that names one block over and over, up to the largest length: the same answer as over the block alone."""
    block = 65536
    g = torch.Generator(device=dev).manual_seed(5)
    k, v = (torch.randn(block, 1, 128, generator=g, device=dev) for _ in range(2))
    args, kval, vval = filled(k, v, "e4m3", block, dev, blocks=1)
    bt = torch.zeros(1, 32768, dtype=torch.int32, device=dev)
    sl = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=dev)
    q = torch.randn(2, 4, 128, generator=g, device=dev).to(torch.bfloat16)
    want = torch.softmax(q.double() @ kval[:, 0].T * SM, -1) @ vval[:, 0]
    # A worker adds 2^31 / 2048 tokens in steps of 32: 2^15 additions of half a step 2^-24 each to the sums of
    # p v and of p, 2 * 2^-9 of the largest value.
    top = float(vval.abs().max())
    lim = bound(top, block, torch.bfloat16, torch.bfloat16, want.cpu().numpy()) + 2.0 ** -8 * top
    got = decode_paged8(q[:1], *args[:4], bt, sl)
    assert np.all((got.double() - want[:1]).abs().cpu().numpy() <= lim[:1])
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    got = prefill_paged8(q, cu, *args[:4], bt, sl)
    assert np.all((got.double() - want).abs().cpu().numpy() <= lim)


def test_tables_without_columns(dev):
    kf, vf = formats("int8", 16)
    kc, vc = (allocate_cache(2, 1, f, device=dev) for f in (kf, vf))
    q = torch.randn(2, 4, 128, device=dev).to(torch.bfloat16)
    bt = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    sl = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    assert not decode_paged8(q, kc, kf, vc, vf, bt, sl).any()
    cu = torch.arange(3, dtype=torch.int32, device=dev)
    assert not prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl).any()


@pytest.mark.parametrize("ranks", [2, 8, 64])
def test_quantize_tokens_between_others(dev, ranks):
    """Every ranks-th token of a prompt has a slot here, the others are another cache's: up to 63 skipped in between."""
    block, n = 16, 40
    kf, vf = formats("e4m3", block)
    blk = [5, 0, 3]
    slots = torch.full((n * ranks,), -1, dtype=torch.int64)
    slots[ranks - 1::ranks] = torch.tensor([blk[i // block] * block + i % block for i in range(n)])
    k, v = (torch.randn(n * ranks, 3, 128, generator=torch.Generator().manual_seed(ranks + i)).to(torch.bfloat16) for i in range(2))
    for cut in (n * ranks, 11 * ranks + 1):    # in one call, and in two that meet inside a block
        caches = [allocate_cache(6, 3, f, device=dev) for f in (kf, vf)]
        want = [ref.Cache(6, 3, block, "e4m3") for _ in range(2)]
        for a, b in ((0, cut), (cut, n * ranks)):
            quantize_paged8_kv(k[a:b].to(dev), v[a:b].to(dev), slots[a:b].to(dev), *caches, kf, vf)
            for w, x in zip(want, (k, v)):
                w.write(x[a:b].double().numpy(), slots[a:b].tolist())
        same_bits(caches[0], want[0], kf)
        same_bits(caches[1], want[1], vf)


def test_calls_side_by_side(dev):
    """Decode and prefill calls on two streams at once: the results of the same calls one after the other."""
    g = torch.Generator(device=dev).manual_seed(9)
    sets = []
    for n in (3001, 700):
        k, v = (torch.randn(n, 2, 128, generator=g, device=dev) for _ in range(2))
        args, _, _ = filled(k, v, "int8", 16, dev)
        q = torch.randn(257, 8, 128, generator=g, device=dev).to(torch.bfloat16)
        cu, sl = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 257], [n]))
        sets.append((q, cu, args, sl))

    def run(s):
        q, cu, args, sl = s
        return prefill_paged8(q, cu, *args, sl), decode_paged8(q[:1], *args, sl)

    want = [run(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for r in got[i]:
            assert torch.equal(r[0], w[0]) and torch.equal(r[1], w[1])


@pytest.mark.parametrize("dtype,seqs,new,hkv,group", [(torch.float32, 8, 2500, 4, 4), (torch.bfloat16, 4, 2048, 8, 4),
                                                      (torch.bfloat16, 64, 130, 8, 4), (torch.float16, 5, 333, 3, 5)])
def test_prefill_prompts(dev, dtype, seqs, new, hkv, group):
    """Prompts of unequal lengths (one of them empty): whole row blocks by tickets, in 32 and 64 rows, and cut ones."""
    g = torch.Generator(device=dev).manual_seed(new)
    block = 16
    lens = [0 if s == 1 else new - 29 * (s % 4) for s in range(seqs)]
    width = -(-new // block)
    kf, vf = formats("e4m3", block)
    kc, vc = (allocate_cache(seqs * width, hkv, f, device=dev) for f in (kf, vf))
    bt = torch.randperm(seqs * width, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev).view(seqs, width)
    for s, n in enumerate(lens):
        t = torch.arange(n, device=dev)
        k, v = (torch.randn(n, hkv, 128, generator=g, device=dev) for _ in range(2))
        quantize_paged8_kv(k, v, bt[s].long()[t // block] * block + t % block, kc, vc, kf, vf)
    starts = np.concatenate([[0], np.cumsum(lens)])
    q = torch.randn(int(starts[-1]), hkv * group, 128, generator=g, device=dev).to(dtype)
    cu, sl = (torch.tensor(np.asarray(x), dtype=torch.int32, device=dev) for x in (starts, lens))
    got = prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=new)
    assert torch.equal(got, prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=new))
    kval, vval = dequantize_paged8(kc, kf).double(), dequantize_paged8(vc, vf).double()
    for s in {0, seqs // 2, seqs - 1}:
        n = lens[s]
        rows = slice(int(starts[s]), int(starts[s + 1]))
        for h in {0, hkv * group - 1}:
            k, v = (x[bt[s].long(), h // group].reshape(-1, 128)[:n] for x in (kval, vval))
            sc = q[rows, h].double() @ k.T.contiguous() * SM
            want = torch.softmax(sc + torch.triu(torch.full_like(sc, -math.inf), diagonal=1), -1) @ v
            lim = bound(float(v.abs().max()), n, dtype, dtype, want.cpu().numpy())
            assert np.all((got[rows, h].double() - want).abs().cpu().numpy() <= lim)


@pytest.mark.parametrize("dtype,seqs,new,past", [(torch.float32, 8, 2500, 0), (torch.bfloat16, 8, 2048, 0), (torch.bfloat16, 3, 333, 0),
                                                 (torch.float16, 2, 200, 9000)])
def test_prefill_nan_changes_nothing_else(dev, dtype, seqs, new, past):
    """NaN against 0 in the same places of V, however the work is dealt: all other outputs keep their bits."""
    g = torch.Generator(device=dev).manual_seed(past + new)
    hkv, group, block, n = 4, 4, 16, past + new
    width = -(-n // block)
    kf, vf = formats("e4m3", block)
    bt = torch.randperm(seqs * width, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(dev).view(seqs, width)
    t = torch.arange(n, device=dev)
    slots = (bt.long()[:, t // block] * block + t % block).reshape(-1)
    k, v = (torch.randn(seqs * n, hkv, 128, generator=g, device=dev) for _ in range(2))
    at = [(s, past + int(f * (new - 1)), h, d) for s, f, h, d in ((0, 0.0, 0, 0), (0, 0.3, 1, 77), (1, 0.77, 3, 127), (seqs - 1, 1.0, 2, 64))]
    outs = []
    q = torch.randn(seqs * new, hkv * group, 128, generator=g, device=dev).to(dtype)
    cu = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device=dev)
    sl = torch.full((seqs,), n, dtype=torch.int32, device=dev)
    for bad in (float("nan"), 0.0):
        for s, p, h, d in at:
            v[s * n + p, h, d] = bad
        kc, vc = (allocate_cache(seqs * width, hkv, f, device=dev) for f in (kf, vf))
        quantize_paged8_kv(k, v, slots, kc, vc, kf, vf)
        outs.append(prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=new))
    want = outs[1].clone().view(seqs, new, hkv, group, 128)
    for s, p, h, d in at:
        want[s, p - past:, h, :, d] = float("nan")
    want = want.view_as(outs[0])
    assert torch.equal(torch.isnan(outs[0]), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(outs[0]), torch.nan_to_num(want))
