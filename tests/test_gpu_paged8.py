"""GPU tests of the 8-bit paged cache: quantisation, decode and prefill attention, against paged8_ref.

Bound of an attention output against 64 bits, per element, with M = max |v| of the case:
  a probability is rounded to fp16 (relative 2^-11; the sum runs over the rounded ones), so an output moves by at
  most 2^-11 max |v_i - out| <= 2^-10 M; one below fp16's normal numbers is off by 2^-25 against a sum of at least
  one: tokens 2^-25 M; a score is an fp32 sum of 128 products, in log2 units off by at most 130 * 2^-24 * sum |q k|,
  which the N(0, 1) inputs keep below 24, and moves the output by at most 2 ln 2 times that: 2^-11.5 M; then the
  output's own rounding.  With f32 on either side the first term is 2^-21 M.
"""

import math

import numpy as np
import pytest
import torch

import paged8_ref as ref
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import (Paged8Format, decode_paged8, dequantize_paged8, prefill_paged8,
                                       quantize_paged8_kv)

pytestmark = pytest.mark.gpu
SM = 1 / math.sqrt(128)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def bound(vmax, tokens, q_dtype, out_dtype, want):
    fine = torch.float32 in (q_dtype, out_dtype)
    return vmax * ((2.0 ** -21 if fine else 2.0 ** -10) + tokens * 2.0 ** -25 + 2.0 ** -11.5) + HALF[out_dtype] * np.abs(want)


def formats(code, block):
    return Paged8Format.for_keys(code, block), Paged8Format.for_values(code, block)


def same_bits(cache, want, fmt):
    """A cache's values against a ref.Cache, NaN for NaN.  (In fp32, which dequantize_paged8 returns: code * scale is exact
    there but where it passes fp32's range, as 256 * 2^120 does for the largest fp32 numbers.)"""
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(dequantize_paged8(cache, fmt).cpu().numpy(), want.values().astype(np.float32))


# ---- quantisation -------------------------------------------------------------------------------

def runs(kind, block, rng):
    """Slots of the calls of a scenario: a list of calls, each a list of slots, in a pool of 24 blocks."""
    blk = rng.permutation(24)
    at = lambda b, r: int(blk[b]) * block + r  # noqa: E731
    seq = lambda b0, a, n: [at(b0 + (a + i) // block, (a + i) % block) for i in range(n)]  # noqa: E731
    if kind == "prompt":
        return [seq(0, 0, 3 * block + 5) + seq(6, 0, 1) + seq(8, 0, block)]
    if kind == "appends":  # one token at a time, two sequences
        return [[at(0, i), at(2, i + 3)] for i in range(min(block - 3, 14))]
    if kind == "extend":   # from the middle of a block on, twice
        return [seq(0, 0, 7) + seq(5, 0, block - 1), seq(0, 7, 2 * block) + seq(5, block - 1, 2), seq(0, 7 + 2 * block, 3)]
    # skipped slots between the others, behind the cache and below zero
    return [[-1] + seq(0, 0, 5) + [24 * block, -7] + seq(0, 5, 3) + [-1, 10 ** 9], [-1, -1]]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block", [16, 48, 128])
@pytest.mark.parametrize("kind", ["prompt", "appends", "extend", "skips"])
def test_quantize_bits(dev, code, dtype, block, kind):
    rng = np.random.default_rng(block + len(kind))
    H = 3
    kf, vf = formats(code, block)
    caches = [allocate_cache(24, H, f, device=dev) for f in (kf, vf)]
    want = [ref.Cache(24, H, block, code) for _ in range(2)]
    for i, slots in enumerate(runs(kind, block, rng)):
        # each call's rows larger than the last one's, by less and by more than a factor of two
        x = [torch.from_numpy(rng.standard_normal((len(slots), H, 128)) * 1.3 ** i * 10.0 ** rng.integers(-3, 3)).to(dtype)
             for _ in range(2)]
        st = torch.tensor(slots, dtype=torch.int64 if i % 2 == 0 else torch.int32, device=dev) if max(slots, default=0) < 2 ** 31 \
            else torch.tensor(slots, dtype=torch.int64, device=dev)
        quantize_paged8_kv(x[0].to(dev), x[1].to(dev), st, caches[0], caches[1], kf, vf)
        for w, y in zip(want, x):
            w.write(y.double().numpy(), slots)
    for c, w, f in zip(caches, want, (kf, vf)):
        same_bits(c, w, f)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_quantize_special_values(dev, code):
    """Zeros, one value, the borders of the scale's steps, ties, the smallest and the largest numbers, infinities, NaN."""
    block, H = 16, 1
    kf, vf = formats(code, block)
    top = ref.TOP[code]
    rows = []
    for vals in ([0.0], [top], [np.nextafter(np.float32(top), np.float32(1e9))], [top * 2.0 ** -10], [1e-45], [2.0 ** -126, 3e-39],
                 [3.4e38, 1.0], [float("inf"), 1.0, -2.0], [float("-inf")], [float("nan"), 5.0], [float("nan")],
                 [top, 0.5, 1.5, 2.5, -0.5, 3.0625, 2.0 ** -7, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -17.0, 18.5]):
        r = np.zeros(128, dtype=np.float32)
        r[5:5 + len(vals)] = vals
        rows.append(r)
    x = np.stack(rows)[:, None]
    T = x.shape[0]
    slots = [i * block for i in range(T)]                       # a block each
    slots2 = [T * block + i for i in range(T)]                  # all in one block, appended one by one
    caches = [allocate_cache(T + 1, H, f, device=dev) for f in (kf, vf)]
    want = ref.Cache(T + 1, H, block, code)
    xt = torch.from_numpy(x).to(dev)
    quantize_paged8_kv(xt, xt, torch.tensor(slots, device=dev), *caches, kf, vf)
    want.write(x.astype(np.float64), slots)
    for i in range(T):
        quantize_paged8_kv(xt[i:i + 1], xt[i:i + 1], torch.tensor([slots2[i]], device=dev), *caches, kf, vf)
        want.write(x[i:i + 1].astype(np.float64), [slots2[i]])
    for c, f in zip(caches, (kf, vf)):
        same_bits(c, want, f)


def test_quantize_restarts_a_block(dev):
    """A block whose first row is written again takes the new rows' scale; a never written block is started by any row."""
    kf, vf = formats("int8", 16)
    caches = [allocate_cache(2, 1, f, device=dev) for f in (kf, vf)]
    x = torch.ones(3, 1, 128, device=dev)
    quantize_paged8_kv(1000 * x[:1], 1000 * x[:1], torch.tensor([0], device=dev), *caches, kf, vf)
    quantize_paged8_kv(x, x, torch.tensor([0, 1, 21], device=dev), *caches, kf, vf)
    for c, f in zip(caches, (kf, vf)):
        got = dequantize_paged8(c, f)
        assert float(c[0, 0, f.code_bytes:f.code_bytes + 4].view(torch.float32)) == 2.0 ** -6
        assert torch.all(got[0, 0, :2] == 1.0) and torch.all(got[1, 0, 5] == 1.0) and torch.all(got[1, 0, 6:] == 0)


def test_quantize_touches_its_tiles_only(dev):
    """Strided, padded caches (K and V halves of one tensor, a spare tail) and strided rows: nothing else changes."""
    kf, vf = formats("e4m3", 16)
    kv = torch.full((5, 3, kf.tile_bytes + vf.tile_bytes + 32), 0xAB, dtype=torch.uint8, device=dev)
    kc, vc = kv[:, :2, :kf.tile_bytes], kv[:, :2, kf.tile_bytes:kf.tile_bytes + vf.tile_bytes]
    kc.zero_()
    vc.zero_()
    big = torch.randn(9, 2, 3, 128, device=dev).to(torch.bfloat16)
    k, v = big[:, 0, :2], big[:, 1, 1:]
    slots = torch.tensor([3 * 16 + i for i in range(9)], device=dev)
    quantize_paged8_kv(k, v, slots, kc, vc, kf, vf)
    want = [ref.Cache(5, 2, 16, "e4m3") for _ in range(2)]
    for w, x in zip(want, (k, v)):
        w.write(x.double().cpu().numpy(), slots.tolist())
    same_bits(kc, want[0], kf)
    same_bits(vc, want[1], vf)
    assert torch.all(kv[:, 2] == 0xAB) and torch.all(kv[:, :, -32:] == 0xAB)
    odd = torch.randn(9 * 2 * 128 + 1, device=dev).to(torch.bfloat16)[1:].view(9, 2, 128)   # off 16-byte alignment
    quantize_paged8_kv(odd, odd, slots, kc, vc, kf, vf)
    want[0].write(odd.double().cpu().numpy(), slots.tolist())
    same_bits(kc, want[0], kf)


def test_quantize_no_tokens(dev):
    kf, vf = formats("e4m3", 16)
    caches = [allocate_cache(2, 2, f, device=dev) for f in (kf, vf)]
    x = torch.zeros(0, 2, 128, device=dev)
    quantize_paged8_kv(x, x, torch.zeros(0, dtype=torch.int64, device=dev), *caches, kf, vf)
    assert not caches[0].any()


# ---- attention -----------------------------------------------------------------------------------

def case(seed, lens, hkv, code, block, spread=0.0, spare=3, hole=False):
    """Caches of random codes over a shuffled pool, tables with garbage behind a sequence's blocks, stale rows (with
    NaN codes) behind its last token."""
    rng = np.random.default_rng(seed)
    kf, vf = formats(code, block)
    need = [-(-n // block) for n in lens]
    n = sum(need) + spare
    perm = rng.permutation(n)
    tables = rng.integers(-5, 2 * n, (len(lens), max(max(need), 1) + 1))
    at, tiles, vals = 0, [], []
    for s, b in enumerate(need):
        tables[s, :b] = perm[at:at + b]
        at += b
        if hole and b > 2:
            tables[s, b // 2] = -1 if s % 2 else n
    for f in (kf, vf):
        scale = 2.0 ** (-7 + np.rint(spread * rng.standard_normal((n, hkv)))) if code == "int8" else \
            2.0 ** (-8 + np.rint(spread * rng.standard_normal((n, hkv))))
        c = ref.codes(rng.standard_normal((n, hkv, block, 128)) * (100 if code == "e4m3" else 40), code)
        tile = ref.pack(c, scale, f)
        vals.append(c * scale[..., None, None])
        tiles.append((tile, f))
    # stale rows: the bytes of an e4m3 NaN (or -1) behind each sequence's end
    off = 0
    for s, ln in enumerate(lens):
        b = need[s]
        if ln % block:
            blk = int(perm[off + b - 1])
            for (tile, f) in tiles:
                body = tile[blk, :, :f.code_bytes].view(hkv, -1)
                rows = torch.arange(ln % block, block)
                if f.layout == "keys":
                    body.view(hkv, block, 128)[:, rows] = 0x7F
                else:
                    body.view(hkv, block // 4, 128, 4)[:, rows // 4, :, rows % 4] = 0x7F
        off += b
    return dict(kf=kf, vf=vf, kc=tiles[0][0], vc=tiles[1][0], kval=vals[0], vval=vals[1],
                bt=torch.from_numpy(tables.astype(np.int32)), lens=torch.tensor(lens, dtype=torch.int32))


def on(c, dev):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def vmax(c):
    return float(np.abs(c["vval"]).max())


def check(got, want, c, tokens, q_dtype):
    g = got.double().cpu().numpy()
    rows = ~np.isnan(want).any(axis=(1, 2))
    err = np.abs(g[rows] - want[rows])
    lim = bound(vmax(c), tokens, q_dtype, got.dtype, want[rows])
    assert np.all(err <= lim), f"worst {np.max(err / lim):.3f} of the bound"
    if torch.float32 in (q_dtype,) and got.dtype == torch.float32 and rows.any():
        # random roundings of 2^-24 steps over 128 products: well below 2^-17 of the values
        assert np.sqrt(np.mean(err ** 2)) <= 2.0 ** -17 * np.sqrt(np.mean(c["vval"] ** 2))


LENS = [37, 1, 0, 16, 17, 300, 33, 2, 64]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group,hkv,block", [(1, 3, 16), (4, 2, 16), (6, 1, 48), (16, 2, 32), (3, 2, 128)])
def test_decode(dev, code, dtype, group, hkv, block):
    c = case(group + block, LENS, hkv, code, block, spread=1.0)
    q = torch.randn(len(LENS), hkv * group, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    d = on(c, dev)
    got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"])
    want = ref.sequences(q.double().numpy(), np.arange(len(LENS) + 1), LENS, c["kval"], c["vval"], c["bt"].numpy(), SM, False, 10 ** 6)
    check(got, want, c, max(LENS), dtype)
    assert torch.all(got[2] == 0)


@pytest.mark.parametrize("lens", [[5000], [4099, 3, 2700], [31] * 200, [1] * 7])
def test_decode_lengths(dev, lens):
    """One long sequence over many waves, ragged ones, many short ones, single tokens."""
    c = case(7, lens, 2, "e4m3", 16)
    q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    d = on(c, dev)
    got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"], max_seq_len=max(lens))
    want = ref.sequences(q.double().numpy(), np.arange(len(lens) + 1), lens, c["kval"], c["vval"], c["bt"].numpy(), SM, False, 10 ** 6)
    check(got, want, c, max(lens), torch.bfloat16)


def test_decode_scales_rising_and_falling(dev):
    """V scales that grow and shrink along a sequence by up to 2^24, K scales that make some tiles' scores dominate."""
    block, lens = 16, [640, 640]
    for dtype in (torch.float16, torch.float32):
        c = case(3, lens, 1, "int8", block)
        kv = c["kval"].copy(), c["vval"].copy()
        for s, sign in enumerate((1, -1)):
            for j in range(40):
                b = int(c["bt"][s, j])
                f = 2.0 ** int(sign * (j - 20) * 0.6)
                kv[1][b] *= f
                for name, val, fmt, g in (("vc", kv[1], c["vf"], f),):
                    at = c[name][b, :, fmt.code_bytes:fmt.code_bytes + 4]
                    at.copy_((at.contiguous().view(torch.float32) * g).view(torch.uint8))
        c["vval"] = kv[1]
        q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(3)).to(dtype)
        d = on(c, dev)
        got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"])
        want = ref.sequences(q.double().numpy(), [0, 1, 2], lens, c["kval"], c["vval"], c["bt"].numpy(), SM, False, 10 ** 6)
        err = np.abs(got.double().cpu().numpy() - want)
        assert np.all(err <= bound(vmax(c), 640, dtype, dtype, want))


@pytest.mark.parametrize("entry", ["decode", "prefill"])
def test_attention_bad_blocks_and_caps(dev, entry):
    """Table entries outside the cache mask their tokens; lengths behind the table (and max_seq_len) are cut."""
    lens = [100, 200, 150]
    c = case(11, lens, 2, "e4m3", 16, hole=True)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(4)).to(torch.float16)
    bt = c["bt"][:, :10].contiguous()             # 160 tokens
    d = on(c, dev)
    if entry == "decode":
        got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], bt.to(dev), d["lens"], max_seq_len=130)
        cap = 130
    else:
        got = prefill_paged8(q.to(dev), torch.arange(4, dtype=torch.int32, device=dev), d["kc"], d["kf"], d["vc"], d["vf"],
                             bt.to(dev), d["lens"])
        cap = 160
    want = ref.sequences(q.double().numpy(), np.arange(4), lens, c["kval"], c["vval"], bt.numpy(), SM, False, cap)
    check(got, want, c, 200, torch.float16)
    gone = torch.full_like(bt, -1).to(dev)
    if entry == "decode":
        got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], gone, d["lens"])
    else:
        got = prefill_paged8(q.to(dev), torch.arange(4, dtype=torch.int32, device=dev), d["kc"], d["kf"], d["vc"], d["vf"], gone, d["lens"])
    assert torch.all(got == 0)


@pytest.mark.parametrize("sm", [-0.05, 0.0, 1.0])
def test_attention_scale(dev, sm):
    """Any finite score scale, negative and zero too; queries far outside fp16's range."""
    lens = [70, 33]
    for entry in ("decode", "prefill"):
        c = case(13, lens, 1, "int8", 16)
        big = 2.0 ** 40
        q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16) * big
        d = on(c, dev)
        if entry == "decode":
            got = decode_paged8(q.to(dev), d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"], sm_scale=sm * SM / big)
        else:
            got = prefill_paged8(q.to(dev), torch.arange(3, dtype=torch.int32, device=dev), d["kc"], d["kf"], d["vc"], d["vf"],
                                 d["bt"], d["lens"], sm_scale=sm * SM / big)
        want = ref.sequences(q.double().numpy(), [0, 1, 2], lens, c["kval"], c["vval"], c["bt"].numpy(), sm * SM / big, False, 10 ** 6)
        check(got, want, c, 70, torch.bfloat16)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group,hkv,block", [(1, 2, 16), (4, 2, 16), (6, 1, 32), (3, 2, 64), (40, 1, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill(dev, code, dtype, group, hkv, block, causal):
    """Ragged sequences: more new tokens than the cache holds (rows that see nothing), none, one, whole prompts, extends."""
    new = [5, 1, 0, 70, 33, 3]
    lens = [37, 1, 9, 70, 333, 2]
    c = case(group + 3 * block, lens, hkv, code, block, spread=1.0)
    starts = np.concatenate([[0], np.cumsum(new)])
    T = int(starts[-1]) + 2                       # two rows of no sequence
    q = torch.randn(T, hkv * group, 128, generator=torch.Generator().manual_seed(6)).to(dtype)
    d = on(c, dev)
    out = torch.full_like(q, 7.0).to(dev)
    got = prefill_paged8(q.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), d["kc"], d["kf"], d["vc"], d["vf"],
                         d["bt"], d["lens"], causal=causal, out=out)
    assert got is out and torch.all(out[T - 2:] == 7.0)
    want = ref.sequences(q.double().numpy(), starts, lens, c["kval"], c["vval"], c["bt"].numpy(), SM, causal, 10 ** 6)
    check(got, want, c, max(lens), dtype)
    if causal:
        assert torch.all(got[int(starts[5])] == 0)   # the first of 3 new tokens in a cache of 2


def rows64(q, d, kval, vval, lens, starts, s, h, group, causal=True):
    """Query rows of sequence s, head h, in 64 bits on the GPU."""
    a, b, L = int(starts[s]), int(starts[s + 1]), lens[s]
    kh = h // group
    block = d["kf"].block_size
    blocks = d["bt"][s, :-(-L // block)].long()
    k = kval[blocks, kh].reshape(-1, 128)[:L]
    v = vval[blocks, kh].reshape(-1, 128)[:L]
    sc = q[a:b, h].double() @ k.T * SM
    if causal:
        sc += torch.triu(torch.full_like(sc, -math.inf), diagonal=L - (b - a) + 1)
    return torch.softmax(sc, -1) @ v


@pytest.mark.parametrize("seqs,new,past,hkv,group", [(8, 1700, 0, 8, 4), (3, 700, 5000, 2, 6), (40, 90, 10, 4, 8), (1, 3000, 0, 1, 3)])
def test_prefill_large(dev, seqs, new, past, hkv, group):
    """Many row blocks (dealt by tickets), few with long keys (cut over several waves), many short ones, one sequence."""
    lens = [past + new - 37 * (s % 3) for s in range(seqs)]
    n_new = [new - 37 * (s % 3) for s in range(seqs)]
    starts = np.concatenate([[0], np.cumsum(n_new)])
    block = 16
    kf, vf = formats("e4m3", block)
    need = [-(-x // block) for x in lens]
    nb = sum(need) + 1
    g = torch.Generator(device=dev).manual_seed(8)
    perm = torch.randperm(nb, generator=g, device=dev).to(torch.int32)
    bt = torch.full((seqs, max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    kc, vc = (allocate_cache(nb, hkv, f, device=dev) for f in (kf, vf))
    for s, b in enumerate(need):
        bt[s, :b] = perm[at:at + b]
        at += b
        slots = (bt[s, :b].long()[:, None] * block + torch.arange(block, device=dev)).reshape(-1)
        x = [torch.randn(b * block, hkv, 128, generator=g, device=dev).to(torch.bfloat16) for _ in range(2)]
        quantize_paged8_kv(x[0], x[1], slots, kc, vc, kf, vf)
    q = torch.randn(int(starts[-1]), hkv * group, 128, generator=g, device=dev).to(torch.float16)
    cu, sl = torch.tensor(starts, dtype=torch.int32, device=dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    got = prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=max(n_new))
    again = prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, max_q_len=max(n_new))
    assert torch.equal(got, again)
    kval, vval = dequantize_paged8(kc, kf).double(), dequantize_paged8(vc, vf).double()
    d = dict(kf=kf, bt=bt)
    for s in {0, seqs // 2, seqs - 1}:
        for h in {0, hkv * group - 1}:
            want = rows64(q, d, kval, vval, lens, starts, s, h, group)
            g64 = got[int(starts[s]):int(starts[s + 1]), h].double()
            lim = bound(float(vval.abs().max()), max(lens), torch.float16, torch.float16, want.cpu().numpy())
            assert np.all((g64 - want).abs().cpu().numpy() <= lim)


def test_attention_nan_stays_in_its_row(dev):
    """A query row that is not finite gives NaN, and no other row does; a NaN value reaches the rows that see it."""
    lens = [50, 700]
    c = case(17, lens, 1, "e4m3", 16)
    d = on(c, dev)
    q = torch.randn(2, 4, 128, device=dev).to(torch.bfloat16)
    q[0, 1, 5], q[1, 2, 7] = float("nan"), float("inf")
    got = decode_paged8(q, d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"])
    bad = torch.isnan(got).all(-1)
    assert bad.tolist() == [[False, True, False, False], [False, False, True, False]] and int(torch.isnan(got).any(-1).sum()) == 2
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    got = prefill_paged8(q, cu, d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"])
    assert torch.equal(torch.isnan(got).all(-1), bad) and int(torch.isnan(got).any(-1).sum()) == 2


def test_attention_destinations(dev):
    """Strided q and out, an out of another type, an out that takes no vector stores."""
    lens = [45, 130]
    c = case(19, lens, 2, "int8", 16)
    d = on(c, dev)
    args = (d["kc"], d["kf"], d["vc"], d["vf"], d["bt"], d["lens"])
    big = torch.randn(2, 12, 256, device=dev).to(torch.bfloat16)
    q = big[:, 2:10, 64:192]
    want = decode_paged8(q.contiguous(), *args)
    strided = torch.zeros(2, 12, 256, dtype=torch.bfloat16, device=dev)
    view = strided[:, 2:10, 64:192]
    assert decode_paged8(q, *args, out=view) is view
    assert torch.equal(view, want) and not strided[:, :2].any() and not strided[:, 10:].any()
    odd = torch.zeros(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 8, 128)
    assert torch.equal(decode_paged8(q, *args, out=odd), want) and torch.equal(odd, want)
    f32 = decode_paged8(q, *args, out=torch.empty(2, 8, 128, device=dev))
    ref64 = ref.sequences(q.double().cpu().numpy(), [0, 1, 2], lens, c["kval"], c["vval"], c["bt"].numpy(), SM, False, 10 ** 6)
    check(f32, ref64, c, 130, torch.bfloat16)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    odd.zero_()
    p = prefill_paged8(q, cu, *args, out=odd)
    check(p, ref64, c, 130, torch.bfloat16)


def test_workspace_given(dev):
    """A caller's workspace: any contents, used as it is; too small or unaligned ones are refused."""
    from turboquant import _lib
    lens = [2000]
    c = on(case(23, lens, 1, "e4m3", 16), dev)
    q = torch.randn(1, 8, 128, device=dev).to(torch.float16)
    args = (c["kc"], c["kf"], c["vc"], c["vf"], c["bt"], c["lens"])
    n = _lib.lib().tq_kv8_decode_workspace_bytes(1, 8, 1)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=dev)
    assert torch.equal(decode_paged8(q, *args, workspace=ws), decode_paged8(q, *args))
    for bad in (ws[:n - 1], ws[1:]):
        with pytest.raises(ValueError):
            decode_paged8(q, *args, workspace=bad)


def test_large_cache_offsets(dev):
    """Blocks beyond 2 GiB of a cache."""
    block, hkv = 16, 8
    kf, vf = formats("e4m3", block)
    nb = (5 << 29) // (hkv * kf.tile_bytes)        # 2.5 GiB each
    kc, vc = (torch.empty(nb, hkv, f.tile_bytes, dtype=torch.uint8, device=dev) for f in (kf, vf))
    ids = [nb - 1, 0, nb - 2, nb // 2]
    x = [torch.randn(60, hkv, 128, device=dev).to(torch.bfloat16) for _ in range(2)]
    slots = torch.tensor([ids[t // block] * block + t % block for t in range(60)], device=dev)
    quantize_paged8_kv(x[0], x[1], slots, kc, vc, kf, vf)
    small = [torch.stack([c[i] for i in ids]) for c in (kc, vc)]
    bt, bs = torch.tensor([ids], dtype=torch.int32, device=dev), torch.arange(4, dtype=torch.int32, device=dev)[None]
    sl = torch.tensor([60], dtype=torch.int32, device=dev)
    q = torch.randn(1, 16, 128, device=dev).to(torch.bfloat16)
    assert torch.equal(decode_paged8(q, kc, kf, vc, vf, bt, sl), decode_paged8(q, small[0], kf, small[1], vf, bs, sl))
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    assert torch.equal(prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl), prefill_paged8(q, cu, small[0], kf, small[1], vf, bs, sl))


def test_side_stream_and_graphs(dev):
    """On a side stream; two captured graphs of the same calls, replayed in turn with new inputs, against eager calls."""
    kf, vf = formats("int8", 16)
    S, hkv, hq = 3, 2, 8
    kc, vc = (allocate_cache(64, hkv, f, device=dev) for f in (kf, vf))
    bt = torch.arange(60, dtype=torch.int32, device=dev).view(3, 20)
    lens = torch.tensor([200, 33, 120], dtype=torch.int32, device=dev)
    for s in range(3):
        n = int(lens[s])
        x = [torch.randn(n, hkv, 128, device=dev) for _ in range(2)]
        quantize_paged8_kv(x[0], x[1], torch.arange(n, device=dev) + 320 * s, kc, vc, kf, vf)
    new = torch.randn(2, S, hkv, 128, device=dev)
    q = torch.randn(S, hq, 128, device=dev)
    slots = torch.zeros(S, dtype=torch.int64, device=dev)
    cu = torch.arange(S + 1, dtype=torch.int32, device=dev)

    def step():
        quantize_paged8_kv(new[0], new[1], slots, kc, vc, kf, vf)
        return decode_paged8(q, kc, kf, vc, vf, bt, lens), prefill_paged8(q, cu, kc, kf, vc, vf, bt, lens, max_q_len=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slots.fill_(-1)
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    slots.fill_(-1)
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for it in range(6):
        g, outs = graphs[it % 2]
        slots.copy_(torch.arange(S, device=dev) * 320 + lens)
        lens += 1
        new.normal_()
        q.normal_()
        keep = kc.clone(), vc.clone()
        g.replay()
        after = kc.clone(), vc.clone()
        got = [o.clone() for o in outs]
        kc.copy_(keep[0])
        vc.copy_(keep[1])
        want = step()
        assert torch.equal(kc, after[0]) and torch.equal(vc, after[1])
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


# ---- refusals on the GPU --------------------------------------------------------------------------

def test_refusals(dev):
    kf, vf = formats("e4m3", 16)
    kc, vc = (allocate_cache(4, 2, f, device=dev) for f in (kf, vf))
    bt = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    sl = torch.ones(1, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 4, 128, device=dev)
    ok = (kc, kf, vc, vf, bt, sl)
    decode_paged8(q, *ok)
    bad = [((q[0],) + ok), ((q[:, :3],) + ok), ((torch.zeros(1, 4, 64, device=dev),) + ok), (torch.zeros(1, 64, 128, device=dev),) + ok,
           (q, vc, vf, kc, kf, bt, sl), (q, kc, kf, vc, Paged8Format.for_values("int8"), bt, sl),
           (q, kc, kf, vc, Paged8Format.for_values("e4m3", 32), bt, sl), (q, kc[:, :1], kf, vc, vf, bt, sl),
           (q, kc[:0], kf, vc[:0], vf, bt, sl), (q, kc[..., :-1], kf, vc, vf, bt, sl), (q, kc, kf, vc, vf, bt[0], sl),
           (q, kc, kf, vc, vf, bt, torch.ones(2, dtype=torch.int32, device=dev))]
    for args in bad:
        with pytest.raises(ValueError):
            decode_paged8(*args)
    for kw in (dict(sm_scale=float("nan")), dict(sm_scale=float("inf")), dict(out=torch.zeros(1, 4, 64, device=dev))):
        with pytest.raises(ValueError):
            decode_paged8(q, *ok, **kw)
    for args in ((q.double(),) + ok, (q, kc, kf, vc, vf, bt.long(), sl), (q, kc, kf, vc, vf, bt, sl.long())):
        with pytest.raises(TypeError):
            decode_paged8(*args)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        prefill_paged8(q, cu.long(), *ok)
    with pytest.raises(ValueError):
        prefill_paged8(q, cu[:1], *ok)
    x = torch.zeros(2, 2, 128, device=dev)
    sm = torch.zeros(2, dtype=torch.int64, device=dev)
    for args in ((x, x[:1], sm), (x[:, :1], x[:, :1], sm), (x, x, sm[:1]), (x[..., :64], x[..., :64], sm)):
        with pytest.raises(ValueError):
            quantize_paged8_kv(*args, kc, vc, kf, vf)
    for args in ((x, x.half(), sm), (x, x, sm.float()), (x.double(), x.double(), sm)):
        with pytest.raises(TypeError):
            quantize_paged8_kv(*args, kc, vc, kf, vf)
