"""GPU tests of windows with sinks over the 8-bit paged cache, and of accumulated weights, against evict8_ref.

Outputs: the bound of test_gpu_paged8.  A weight is exp(s - M) / l in fp32: a score is an fp32 sum of 128 products and three
more roundings, in log2 units off by at most 131 * 2^-24 * sum |q k|, which the N(0, 1) inputs keep below 24; in 16 bits the
query is exact but for elements below 2^-16 of the row's largest, which are off by 2^-25 of at most four times their unit: 128 *
2^-23 of the largest |k| (below 2^3) against scores of the same kind, 2^-13 in all; f32 queries keep 2^-22 of each
element, below the sums' roundings.  A weight moves by ln 2 times its score's error and once more by its row's sum, by
2^-22 for the exponential and by 2^-24 for each rounding of a sum (tokens / 16 in one lane, then the lanes, 24).
"""

import math

import numpy as np
import pytest
import torch

import evict8_ref as eref
from test_gpu_paged8 import SM, bound, formats
from turboquant.kernels.evict8 import allocate_mass, observe_paged8
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import decode_paged8, dequantize_paged8, prefill_paged8, quantize_paged8_kv

pytestmark = pytest.mark.gpu


def weight_error(tokens, rows):
    """Relative to the sum of the weights that were added."""
    score = 131 * 2.0 ** -24 * 24 + 2.0 ** -13
    return 2 * math.log(2) * score + 2.0 ** -22 + (tokens / 16 + 24 + rows) * 2.0 ** -24


def caches(dev, lens, hkv, code, block, seed=0, width=None, extra=3, kv=None):
    """Caches that hold sequences of the given lengths in shuffled blocks: (kc, kf, vc, vf, tables), their values."""
    g = torch.Generator(device=dev).manual_seed(seed)
    kf, vf = formats(code, block)
    need = [-(-n // block) for n in lens]
    kc, vc = (allocate_cache(sum(need) + extra, hkv, f, device=dev) for f in (kf, vf))
    perm = torch.randperm(kc.shape[0], generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    bt = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
    slots, at = [], 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
        t = torch.arange(lens[s])
        slots.append(bt[s, t // block].long() * block + t % block)
    slots = torch.cat(slots).to(dev)
    k, v = kv if kv is not None else (torch.randn(sum(lens), hkv, 128, generator=g, device=dev) for _ in range(2))
    quantize_paged8_kv(k, v, slots, kc, vc, kf, vf)
    return (kc, kf, vc, vf, bt.to(dev)), [dequantize_paged8(c, f).cpu().double().numpy() for c, f in ((kc, kf), (vc, vf))]


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def random_mass(kc, block, seed=5):
    return torch.rand(kc.shape[0], kc.shape[1], block, generator=torch.Generator().manual_seed(seed)).to(kc.device)


def check_mass(got, before, want_add, tables, lens, new, block, rows, label=""):
    want = before.cpu().double().numpy().copy()
    tol = np.abs(want) * 2.0 ** -24
    for s, L in enumerate(lens):
        if new[s] or want_add[s] is not None:
            eref.accumulate(want, want_add[s], tables[s], L, new[s], block)
            for t in range(L):
                b = int(tables[s][t // block])
                if 0 <= b < want.shape[0]:
                    a = want_add[s][:, t]
                    tol[b, :, t % block] = a * weight_error(L, rows) + np.abs(want[b, :, t % block]) * 2.0 ** -23 + 2.0 ** -126
    err = np.abs(got.cpu().double().numpy() - want)
    assert np.all(err <= tol), (label, np.max(err / np.maximum(tol, 1e-300)))


WINDOWS = [(1, 0), (1, 1), (16, 0), (33, 4), (31, 40), (100, 16), (500, 130), (1 << 40, 7)]


@pytest.mark.parametrize("code,qd,block", [("e4m3", torch.bfloat16, 16), ("int8", torch.float16, 48), ("e4m3", torch.float32, 32),
                                           ("int8", torch.float32, 16)])
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_decode(dev, code, qd, block, window, sinks):
    lens = [0, 1, 2, 15, 16, 17, 32, 33, 64, 100, 131, 260, 517, 1300]
    hkv, group = 2, 3
    args, (kval, vval) = caches(dev, lens, hkv, code, block, seed=window % 97 + sinks)
    q = torch.randn(len(lens), hkv * group, 128, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(qd)
    before = random_mass(args[0], block)
    mass = before.clone()
    kc, kf, vc, vf, bt = args
    sl = i32(lens, dev)
    out = decode_paged8(q, kc, kf, vc, vf, bt, sl, window=window, sinks=sinks)
    both = decode_paged8(q, kc, kf, vc, vf, bt, sl, window=window, sinks=sinks, mass=mass, max_seq_len=1300)
    adds = []
    for s, L in enumerate(lens):
        w, add = eref.sequence(q[s:s + 1].cpu().double().numpy(), kval, vval, bt[s].cpu(), L, window, sinks, SM)
        adds.append(add)
        if not L:
            w[:] = 0
        for o in (out, both):
            err = np.abs(o[s].cpu().double().numpy() - w[0])
            assert np.all(err <= bound(np.abs(vval).max(), L, qd, qd, w[0])), (L, err.max())
    check_mass(mass, before, adds, bt.cpu(), lens, [min(L, 1) for L in lens], block, 1)


@pytest.mark.parametrize("code,qd,group,window,sinks", [("e4m3", torch.bfloat16, 1, None, 0), ("int8", torch.float16, 16, None, 0),
                                                        ("e4m3", torch.float32, 16, 8000, 40), ("int8", torch.bfloat16, 1, 6000, 0)])
def test_mass_of_many_pieces(dev, code, qd, group, window, sinks):
    """A segment shared by more waves than a wave has lanes (at least two steps of 32 tokens each), one and sixteen query heads to it.

    (A row's sum is then at most five tokens' in a lane and nine joins of four roundings, less than the tokens / 16 that
    weight_error counts.)"""
    lens = [9000, 0, 700]
    args, (kval, vval) = caches(dev, lens, 1, code, 16, seed=group)
    kc, kf, vc, vf, bt = args
    q = torch.randn(3, group, 128, generator=torch.Generator(device=dev).manual_seed(5), device=dev).to(qd)
    before = random_mass(kc, 16)
    mass = before.clone()
    out = decode_paged8(q, *args, i32(lens, dev), window=window, sinks=sinks, mass=mass)
    adds = []
    for s, L in enumerate(lens):
        want, add = eref.sequence(q[s:s + 1].cpu().double().numpy(), kval, vval, bt[s].cpu(), L, window, sinks, SM) if L else (
            np.zeros((1, group, 128)), np.zeros((1, 0)))
        adds.append(add)
        assert np.all(np.abs(out[s].cpu().double().numpy() - want[0]) <= bound(np.abs(vval).max(), L, qd, qd, want[0]))
    check_mass(mass, before, adds, bt.cpu(), lens, [1, 0, 1], 16, group)


@pytest.mark.parametrize("code,qd,block", [("e4m3", torch.bfloat16, 16), ("int8", torch.float16, 48), ("e4m3", torch.float32, 64)])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("group", [1, 5])
def test_prefill(dev, code, qd, block, window, sinks, group):
    new = [1, 0, 40, 7, 150, 65, 3]
    past = [0, 20, 0, 300, 77, 500, 31]
    lens = [p + n for p, n in zip(past, new)]
    hkv = 2
    args, (kval, vval) = caches(dev, lens, hkv, code, block, seed=window % 89 + sinks)
    T = sum(new)
    q = torch.randn(T + 2, hkv * group, 128, generator=torch.Generator(device=dev).manual_seed(2), device=dev).to(qd)
    at = np.concatenate([[0], np.cumsum(new)])
    out = torch.full_like(q, 7.0)
    prefill_paged8(q, i32(at, dev), *args, i32(lens, dev), max_q_len=150, out=out, window=window, sinks=sinks)
    assert torch.all(out[T:] == 7.0)                                            # rows of no sequence
    for s, L in enumerate(lens):
        a, b = at[s], at[s + 1]
        want, _ = eref.sequence(q[a:b].cpu().double().numpy(), kval, vval, args[4][s].cpu(), L, window, sinks, SM)
        err = np.abs(out[a:b].cpu().double().numpy() - want)
        assert np.all(err <= bound(np.abs(vval).max(), L, qd, qd, want)), (s, err.max())


@pytest.mark.parametrize("code,qd", [("e4m3", torch.bfloat16), ("int8", torch.float32)])
@pytest.mark.parametrize("seqs,new,past,window,sinks", [(1, 900, 3000, 700, 4), (3, 1500, 0, 200, 64), (40, 64, 128, 90, 5),
                                                        (2, 2000, 10, 64, 0)])
def test_prefill_dealings(dev, code, qd, seqs, new, past, window, sinks):
    """The ways in which a call is dealt to the device's waves: rows against the unwindowed kernel on the tokens they see."""
    news = [new - 3 * (s % 20) for s in range(seqs)]
    lens = [past + n for n in news]
    args, (kval, vval) = caches(dev, lens, 1, code, 16, seed=seqs)
    T = sum(news)
    q = torch.randn(T, 4, 128, generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(qd)
    at = np.concatenate([[0], np.cumsum(news)])
    out = prefill_paged8(q, i32(at, dev), *args, i32(lens, dev), window=window, sinks=sinks)
    again = prefill_paged8(q, i32(at, dev), *args, i32(lens, dev), window=window, sinks=sinks)
    assert torch.equal(out, again)
    kt, vt = (torch.from_numpy(x).to(dev) for x in (kval, vval))
    for s, L in enumerate(lens):
        t = torch.arange(L, device=dev)
        blk = args[4][s][t // 16].long()
        k, v = kt[blk, 0, t % 16], vt[blk, 0, t % 16]
        p = torch.arange(L - news[s], L, device=dev)[:, None]
        see = (t[None] <= p) & ((t[None] > p - window) | (t[None] < sinks))
        for h in range(4):
            sc = torch.where(see, q[at[s]:at[s + 1], h].double() @ k.T * SM, -math.inf)
            want = (torch.softmax(sc, 1) @ v).cpu().numpy()
            err = np.abs(out[at[s]:at[s + 1], h].cpu().double().numpy() - want)
            assert np.all(err <= bound(np.abs(vval).max(), L, qd, qd, want)), (s, h, err.max())


def test_window_of_all_tokens_is_none(dev):
    """A window as long as the sequence, or sinks that meet it, see what an unwindowed call sees."""
    lens = [700, 40, 333]
    args, _ = caches(dev, lens, 2, "e4m3", 16)
    q = torch.randn(3, 8, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    sl, cu = i32(lens, dev), i32([0, 1, 2, 3], dev)
    want, wantp = decode_paged8(q, *args, sl), prefill_paged8(q, cu, *args, sl)
    for w, sinks in ((700, 0), (1 << 31, 0), (300, 400), (1, 699)):
        # (f32: probabilities of 22 bits; the cuts between waves differ)
        assert torch.allclose(decode_paged8(q, *args, sl, window=w, sinks=sinks), want, rtol=0, atol=2.0 ** -17)
        assert torch.allclose(prefill_paged8(q, cu, *args, sl, window=w, sinks=sinks), wantp, rtol=0, atol=2.0 ** -17)


@pytest.mark.parametrize("window,sinks", [(40, 0), (40, 5), (70, 33)])
@pytest.mark.parametrize("qd", [torch.bfloat16, torch.float32])
def test_nan_outside_the_window(dev, window, sinks, qd):
    """NaN of K or V reaches the rows that see its token, in its dims, and no others."""
    L, new = 300, 90
    g = torch.Generator(device=dev).manual_seed(window)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    bad = {3: 1, 100: 2, 180: 3, 215: 4, 250: 5, 299: 6}
    for t, d in bad.items():
        v[t, 0, d] = float("nan")
    k[5, 0, 9] = k[L - 60, 0, 9] = float("nan")
    args, (kval, vval) = caches(dev, [L], 1, "e4m3", 16, kv=(k, v))
    q = torch.randn(new, 3, 128, generator=g, device=dev).to(qd)
    out = prefill_paged8(q, i32([0, new], dev), *args, i32([L], dev), window=window, sinks=sinks).cpu().double().numpy()
    single = [decode_paged8(q[i:i + 1], *args, i32([L - new + 1 + i], dev), window=window, sinks=sinks).cpu().double().numpy()[0]
              for i in range(0, new, 11)]
    clean = [np.nan_to_num(x, nan=0.0) for x in (kval, vval)]
    want, _ = eref.sequence(q.cpu().double().numpy(), *clean, args[4][0].cpu(), L, window, sinks, SM)
    for i in range(new):
        see = eref.visible(L - new + i, L, window, sinks)
        nan = np.zeros(128, dtype=bool)
        for t, d in bad.items():
            nan[d] |= bool(see[t])
        if see[5] or see[L - 60]:
            nan[:] = True
        for o in [out[i]] + ([single[i // 11]] if i % 11 == 0 else []):
            for h in range(3):
                np.testing.assert_array_equal(np.isnan(o[h]), nan)
                ok = ~nan
                assert np.all(np.abs(o[h] - want[i, h])[ok] <= bound(8.0, L, qd, qd, want[i, h])[ok])


def test_far_scales_outside_the_window(dev):
    """Values 2^60 times larger behind the window do not touch what is seen."""
    L, W = 400, 50
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    v[:L - 120] *= 2.0 ** 60
    args, (kval, vval) = caches(dev, [L], 1, "int8", 16, kv=(k, v))
    q = torch.randn(64, 2, 128, generator=g, device=dev).to(torch.bfloat16)
    out = prefill_paged8(q, i32([0, 64], dev), *args, i32([L], dev), window=W)
    one = decode_paged8(q[-1:], *args, i32([L], dev), window=W)
    want, _ = eref.sequence(q.cpu().double().numpy(), kval, vval, args[4][0].cpu(), L, W, 0, SM)
    # (the first row's window begins with token 287, the last of the block 272..287, whose scale is 2^60 times that of the blocks
    # behind it: those count as zeros for it, by the documented 2^-24, and token 287 itself was quantised to zeros)
    want[0] = 0.0
    assert L - 64 - W + 1 == 287 and not vval[int(args[4][0, 17])][0, 15].any()
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= bound(8.0, L, q.dtype, q.dtype, want))
    assert np.all(np.abs(one.cpu().double().numpy() - want[-1:]) <= bound(8.0, L, q.dtype, q.dtype, want[-1:]))


def test_bad_blocks_and_cut_lengths(dev):
    """Table entries outside the cache mask their tokens; max_seq_len cuts; tables wider than needed."""
    lens = [200, 333, 64]
    args, (kval, vval) = caches(dev, lens, 2, "e4m3", 16, width=30)
    kc, kf, vc, vf, bt = args
    bt[0, 3], bt[0, 11], bt[1, 20], bt[2] = -1, 10 ** 6, -7, -1
    q = torch.randn(3, 4, 128, generator=torch.Generator(device=dev).manual_seed(8), device=dev).to(torch.float16)
    before = random_mass(kc, 16)
    mass = before.clone()
    out = decode_paged8(q, kc, kf, vc, vf, bt, i32([200, 999, 64], dev), max_seq_len=333, window=100, sinks=20, mass=mass)
    adds = []
    for s, L in enumerate(lens):
        want, add = eref.sequence(q[s:s + 1].cpu().double().numpy(), kval, vval, bt[s].cpu(), L, 100, 20, SM)
        adds.append(add)
        assert np.all(np.abs(out[s].cpu().double().numpy() - want[0]) <= bound(np.abs(vval).max(), L, q.dtype, q.dtype, want[0]))
    check_mass(mass, before, adds, bt.cpu(), lens, [1, 1, 1], 16, 1)
    assert not out[2].any()


@pytest.mark.parametrize("code,qd,block,window,sinks,last", [
    ("e4m3", torch.bfloat16, 16, None, 0, None), ("int8", torch.float16, 48, None, 0, 5), ("e4m3", torch.float32, 32, 50, 3, 70),
    ("int8", torch.float32, 16, 1, 0, 1), ("e4m3", torch.bfloat16, 64, 90, 100, 33), ("int8", torch.bfloat16, 16, 300, 0, None)])
@pytest.mark.parametrize("group", [1, 3, 16])
def test_observe(dev, code, qd, block, window, sinks, last, group):
    new = [1, 0, 40, 7, 150, 65]
    past = [0, 20, 0, 300, 77, 600]
    lens = [p + n for p, n in zip(past, new)]
    hkv = 2
    args, (kval, vval) = caches(dev, lens, hkv, code, block, seed=group)
    kc, kf, _, _, bt = args
    q = torch.randn(sum(new) + 3, hkv * group, 128, generator=torch.Generator(device=dev).manual_seed(6), device=dev).to(qd)
    at = np.concatenate([[0], np.cumsum(new)])
    before = random_mass(kc, block)
    mass = before.clone()
    got = observe_paged8(q, i32(at, dev), kc, kf, bt, i32(lens, dev), mass, last=last, window=window, sinks=sinks)
    assert got is mass
    adds = [eref.sequence(q[at[s]:at[s + 1]].cpu().double().numpy(), kval, None, bt[s].cpu(), L, window, sinks, SM, last)[1]
            if new[s] else None for s, L in enumerate(lens)]
    rows = group * min(150, last or 150)
    check_mass(mass, before, adds, bt.cpu(), lens, new, block, rows)


@pytest.mark.parametrize("window", [None, 700])
def test_observe_long(dev, window):
    """Many row blocks and many chunks of keys; the same call gives the same bits."""
    new, past = [1000, 30], [500, 9000]
    lens = [p + n for p, n in zip(past, new)]
    args, (kval, _) = caches(dev, lens, 1, "e4m3", 16)
    kc, kf, _, _, bt = args
    q = torch.randn(sum(new), 4, 128, generator=torch.Generator(device=dev).manual_seed(6), device=dev).to(torch.bfloat16)
    before = random_mass(kc, 16)
    got = [observe_paged8(q, i32([0, 1000, 1030], dev), kc, kf, bt, i32(lens, dev), before.clone(), window=window) for _ in range(2)]
    assert torch.equal(*got)
    adds, at = [], 0
    for s, L in enumerate(lens):
        t = torch.arange(L, device=dev)
        k = torch.from_numpy(kval).to(dev)[bt[s][t // 16].long(), 0, t % 16]
        p = torch.arange(past[s], L, device=dev)[:, None]
        see = (t[None] <= p) & (t[None] > p - (window or L))
        add = sum(torch.softmax(torch.where(see, q[at:at + new[s], h].double() @ k.T * SM, -math.inf), 1).sum(0) for h in range(4))
        adds.append(add[None].cpu().numpy())
        at += new[s]
    check_mass(got[0], before, adds, bt.cpu(), lens, new, 16, 4000)


def test_weights_that_are_not_numbers(dev):
    """A NaN in a key or a query takes the weights of the rows that see it, and no others, out of the sums."""
    L, new = 120, 50
    g = torch.Generator(device=dev).manual_seed(12)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    k[95, 0, 3] = float("nan")
    args, (kval, vval) = caches(dev, [L], 1, "e4m3", 16, kv=(k, v))
    kc, kf, vc, vf, bt = args
    q = torch.randn(new, 2, 128, generator=g, device=dev)
    q[4, 1, 77] = float("nan")
    q[9, 0, 5] = float("inf")
    before = random_mass(kc, 16)
    got = observe_paged8(q, i32([0, new], dev), kc, kf, bt, i32([L], dev), before.clone())
    add = np.zeros((1, L))
    for i in range(new):
        for h in range(2):
            see = eref.visible(L - new + i, L, None, 0)
            if not see[95] and not (i, h) in ((4, 1), (9, 0)):
                add[0] += eref.weights(q[i, h].cpu().double().numpy(), np.nan_to_num(eref.ref.gather(kval, bt[0].cpu(), L)[0][:, 0]), see, SM)
    check_mass(got, before, [add], bt.cpu(), [L], [new], 16, 2 * new)
    # decode: the last token alone starts from 0, the others keep their numbers
    mass = before.clone()
    out = decode_paged8(q[:1], kc, kf, vc, vf, bt, i32([L], dev), mass=mass)
    assert out.isnan().all()
    check_mass(mass, before, [np.zeros((1, L))], bt.cpu(), [L], [1], 16, 1)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("qd,heads", [(torch.bfloat16, 2), (torch.float32, 1)])
def test_far_query_among_ordinary_ones(dev, qd, heads, first):
    """A query whose scores pass fp32's range adds nothing and takes nothing from the rows that share its lanes.

    Its |q| of 3e38 takes a factor of 2^126 or more, and keys of some thousands a scale of 2^5 or more, 2^-3 for the softmax's own: the
    product passes 2^128.  Ordinary queries are 2^-12 of N(0, 1), so that their scores are those of N(0, 1) rows.  first: it is the
    call's first row, whose factor rows of padding would take over."""
    L, new, size = 300, 150, 2.0 ** -12
    g = torch.Generator(device=dev).manual_seed(heads)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    args, (kval, _) = caches(dev, [L], 1, "int8", 16, kv=(k / size, v))
    kc, kf, _, _, bt = args
    q = (torch.randn(new, heads, 128, generator=g, device=dev) * size).to(qd)
    at = 0 if first else 37
    q[at, 0] = torch.where(torch.rand(128, generator=g, device=dev) < 0.5, -3e38, 3e38).to(qd)
    assert q.isfinite().all()
    before = random_mass(kc, 16)
    got = observe_paged8(q, i32([0, new], dev), kc, kf, bt, i32([L], dev), before.clone())
    keys = eref.ref.gather(kval, bt[0].cpu(), L)[0][:, 0]
    add = np.zeros((1, L))
    for i in range(new):
        for h in range(heads):
            if (i, h) != (at, 0):
                add[0] += eref.weights(q[i, h].cpu().double().numpy(), keys, eref.visible(L - new + i, L, None, 0), SM)
    check_mass(got, before, [add], bt.cpu(), [L], [new], 16, heads * new)


def test_observe_short_sequences(dev):
    """More queries than tokens (rows before the sequence's start see nothing), lengths of 0 and 1, cut lengths."""
    args, (kval, _) = caches(dev, [30, 1, 64], 1, "int8", 16, width=5)
    kc, kf, _, _, bt = args
    q = torch.randn(60, 2, 128, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.float16)
    before = random_mass(kc, 16)
    mass = before.clone()
    observe_paged8(q, i32([0, 40, 40, 45, 60], dev), kc, kf, torch.cat([bt, bt[:1]])[[0, 1, 1, 2]].contiguous(), i32([30, 0, 1, 999], dev), mass,
                   max_seq_len=64)
    adds = []
    for s, (L, a, b) in enumerate(((30, 0, 40), (1, 40, 45), (64, 45, 60))):
        add = np.zeros((1, L))
        k = eref.ref.gather(kval, bt[s].cpu(), L)[0][:, 0]
        for i in range(b - a):
            p = L - (b - a) + i
            for h in range(2):
                add[0] += eref.weights(q[a + i, h].cpu().double().numpy(), k, eref.visible(p, L, None, 0), SM)
        adds.append(add)
    check_mass(mass, before, adds, bt.cpu(), [30, 1, 64], [40, 5, 15], 16, 80)


def test_strided_and_other_stream(dev):
    """Strided queries, tables, mass and caches, on a stream of their own."""
    lens = [150, 333]
    args, (kval, vval) = caches(dev, lens, 2, "e4m3", 16)
    kc, kf, vc, vf, bt = args
    big = torch.zeros(kc.shape[0], 5, 2 * kc.shape[2], dtype=torch.uint8, device=dev)
    big[:, 1:3, :kc.shape[2]], big[:, 1:3, kc.shape[2]:] = kc, vc
    kc2, vc2 = big[:, 1:3, :kc.shape[2]], big[:, 1:3, kc.shape[2]:]
    wide = torch.full((2, 60), -5, dtype=torch.int32, device=dev)
    wide[:, :bt.shape[1]] = bt
    before = random_mass(kc, 16)
    mass = torch.zeros(kc.shape[0], 3, 24, device=dev)
    mass[:, :2, :16] = before
    view = mass[:, :2, :16]
    q = torch.randn(2, 260, 6, generator=torch.Generator(device=dev).manual_seed(3), device=dev).to(torch.bfloat16).transpose(1, 2)[..., 1:129]
    sl = i32([150, 0, 333, 0], dev)[::2]
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        out = decode_paged8(q, kc2, kf, vc2, vf, wide[:, :bt.shape[1]], sl, window=90, sinks=3, mass=view)
        cu = i32([0, 1, 2], dev)
        out2 = prefill_paged8(q, cu, kc2, kf, vc2, vf, wide[:, :bt.shape[1]], sl, window=90, sinks=3)
        view2 = torch.zeros(kc.shape[0], 3, 24, device=dev)[:, :2, :16]
        view2.copy_(before)
        observe_paged8(q, cu, kc2, kf, wide[:, :bt.shape[1]], sl, view2, window=90, sinks=3)
    torch.cuda.current_stream(dev).wait_stream(stream)
    adds = []
    for s, L in enumerate(lens):
        want, add = eref.sequence(q[s:s + 1].cpu().double().numpy(), kval, vval, bt[s].cpu(), L, 90, 3, SM)
        adds.append(add)
        for o in (out, out2):
            assert np.all(np.abs(o[s].cpu().double().numpy() - want[0]) <= bound(np.abs(vval).max(), L, q.dtype, q.dtype, want[0]))
    for m in (view, view2):
        check_mass(m, before, adds, bt.cpu(), lens, [1, 1], 16, 1)
    assert not mass[:, 2].any() and not mass[..., 16:].any()


def test_refusals(dev):
    args, _ = caches(dev, [40, 20], 2, "e4m3", 16)
    kc, kf, vc, vf, bt = args
    q, sl, cu = torch.randn(2, 4, 128, device=dev), i32([40, 20], dev), i32([0, 1, 2], dev)
    mass = allocate_mass(kc.shape[0], 2, 16, device=dev)
    for kw in (dict(window=0), dict(window=-3), dict(sinks=2), dict(window=4, sinks=-1), dict(mass=mass[:-1]), dict(mass=mass.double()),
               dict(mass=mass.cpu()), dict(mass=mass[..., :8]), dict(mass=mass[:, :1].expand(-1, 2, -1)),
               dict(mass=mass, workspace=torch.empty(256, dtype=torch.uint8, device=dev))):
        with pytest.raises(ValueError):
            decode_paged8(q, *args, sl, **kw)
    for kw in (dict(window=0), dict(sinks=2), dict(window=4, sinks=-1), dict(window=4, causal=False)):
        with pytest.raises(ValueError):
            prefill_paged8(q, cu, *args, sl, **kw)
    good = dict(q=q, cu_seqlens_q=cu, k_cache=kc, k_fmt=kf, block_tables=bt, seq_lens=sl, mass=mass)
    for kw in (dict(last=0), dict(last=-1), dict(window=0), dict(sinks=1), dict(q=q[0]), dict(q=q[..., :64]), dict(q=q[:, :3]),
               dict(cu_seqlens_q=cu[:-1]), dict(k_fmt=vf), dict(k_cache=kc[..., :-16]), dict(k_cache=kc.float()), dict(seq_lens=sl[:1]),
               dict(block_tables=bt[:, ::2]), dict(mass=mass[..., :8]), dict(sm_scale=float("nan")), dict(sm_scale=float("inf")),
               dict(workspace=torch.empty(16, dtype=torch.uint8, device=dev)), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            observe_paged8(**{**good, **kw})
    for kw in (dict(cu_seqlens_q=cu.long()), dict(seq_lens=sl.long()), dict(block_tables=bt.long()), dict(q=q.double())):
        with pytest.raises(TypeError):
            observe_paged8(**{**good, **kw})
    before = mass.clone()
    observe_paged8(**{**good, "q": q[:0], "cu_seqlens_q": i32([0, 0, 0], dev)})
    observe_paged8(**{**good, "max_q_len": 0})
    assert torch.equal(mass, before)


@pytest.mark.parametrize("sm", [0.0, -0.06, 0.02])
@pytest.mark.parametrize("qd", [torch.bfloat16, torch.float32])
def test_score_scales(dev, sm, qd):
    """No scale (all tokens alike), a negative one, a small one."""
    L, new = 300, 20
    args, (kval, vval) = caches(dev, [L], 2, "int8", 16)
    kc, kf, vc, vf, bt = args
    q = torch.randn(new, 4, 128, generator=torch.Generator(device=dev).manual_seed(4), device=dev).to(qd)
    before = random_mass(kc, 16)
    got = observe_paged8(q, i32([0, new], dev), kc, kf, bt, i32([L], dev), before.clone(), sm_scale=sm, window=120, sinks=2)
    _, add = eref.sequence(q.cpu().double().numpy(), kval, None, bt[0].cpu(), L, 120, 2, sm)
    check_mass(got, before, [add], bt.cpu(), [L], [new], 16, 2 * new)
    mass = before.clone()
    out = decode_paged8(q[-1:], *args, i32([L], dev), sm_scale=sm, window=120, sinks=2, mass=mass)
    want, add = eref.sequence(q[-1:].cpu().double().numpy(), kval, vval, bt[0].cpu(), L, 120, 2, sm)
    check_mass(mass, before, [add], bt.cpu(), [L], [1], 16, 2)
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= bound(np.abs(vval).max(), L, qd, qd, want))


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 14, 2.0 ** 30])
def test_far_scores(dev, size):
    """Scores so large that fp32's spacing passes one unit: every row's weights still are numbers and sum to one."""
    L, new, hq = 500, 70, 4
    g = torch.Generator(device=dev).manual_seed(11)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    args, _ = caches(dev, [L], 1, "e4m3", 16, kv=(k * size, v))
    kc, kf, vc, vf, bt = args
    q = torch.randn(new, hq, 128, generator=g, device=dev) * size
    mass = observe_paged8(q, i32([0, new], dev), kc, kf, bt, i32([L], dev), allocate_mass(kc.shape[0], 1, 16, device=dev))
    one = allocate_mass(kc.shape[0], 1, 16, device=dev)
    decode_paged8(q[-1:], *args, i32([L], dev), mass=one)
    # (L weights of a row and their sum: two roundings each, an exponential of 2^-22 on either side)
    for m, rows in ((mass, new * hq), (one, hq)):
        assert torch.all(m >= 0) and abs(m.double().sum().item() - rows) <= rows * (2.0 ** -21 + (L + rows) * 2.0 ** -24)


@pytest.mark.parametrize("code,qd", [("e4m3", torch.float32), ("int8", torch.bfloat16), ("e4m3", torch.float16), ("int8", torch.float32)])
@pytest.mark.parametrize("window,sinks,group", [(37, 3, 2), (20, 0, 1), (70, 17, 5)])
def test_scales_by_block(dev, code, qd, window, sinks, group):
    """Blocks whose values differ by 2^40: a row is as exact as the blocks that it sees allow, whatever others hold."""
    L, new = 700, 200
    g = torch.Generator(device=dev).manual_seed(window)
    k, v = (torch.randn(L, 1, 128, generator=g, device=dev) for _ in range(2))
    e = torch.randint(-1, 2, (-(-L // 16),), generator=torch.Generator().manual_seed(window)).to(dev).double() * 40
    v = (v.double() * torch.exp2(e)[torch.arange(L, device=dev) // 16][:, None, None]).float()
    args, (kval, vval) = caches(dev, [L], 1, code, 16, kv=(k, v))
    q = torch.randn(new, group, 128, generator=g, device=dev).to(qd)
    out = torch.empty(new, group, 128, device=dev, dtype=torch.float32 if qd == torch.float16 else qd)  # (2^40 is no half)
    prefill_paged8(q, i32([0, new], dev), *args, i32([L], dev), window=window, sinks=sinks, out=out)
    want, _ = eref.sequence(q.cpu().double().numpy(), kval, vval, args[4][0].cpu(), L, window, sinks, SM)
    got = out.cpu().double().numpy()
    for i in range(new):
        seen = np.nonzero(eref.visible(L - new + i, L, window, sinks))[0]
        # (a block's scale holds for all its rows, so what counts is the largest that its codes could be)
        top = max(np.abs(vval[int(args[4][0, b])]).max() for b in set(seen // 16)) * 2
        assert np.all(np.abs(got[i] - want[i]) <= bound(top, L, qd, out.dtype, want[i])), i


@pytest.mark.parametrize("group", [17, 70, 130])
def test_many_heads(dev, group):
    """More query heads per KV head than a row block's share: prefill with a window, and prompts' weights."""
    lens, new, block = [90, 200], [5, 11], 16
    args, (kval, vval) = caches(dev, lens, 1, "e4m3", block)
    q = torch.randn(16, group, 128, generator=torch.Generator(device=dev).manual_seed(group), device=dev).to(torch.bfloat16)
    cu, sl = i32([0, 5, 16], dev), i32(lens, dev)
    out = prefill_paged8(q, cu, *args, sl, window=50, sinks=3)
    before = random_mass(args[0], block)
    mass = observe_paged8(q, cu, args[0], args[1], args[4], sl, before.clone(), last=4, window=50, sinks=3)
    adds = []
    for s, (a, b) in enumerate(((0, 5), (5, 16))):
        want, add = eref.sequence(q[a:b].cpu().double().numpy(), kval, vval, args[4][s].cpu(), lens[s], 50, 3, SM, 4)
        adds.append(add)
        assert np.all(np.abs(out[a:b].cpu().double().numpy() - want) <= bound(np.abs(vval).max(), lens[s], q.dtype, q.dtype, want))
    check_mass(mass, before, adds, args[4].cpu(), lens, new, block, 4 * group)
