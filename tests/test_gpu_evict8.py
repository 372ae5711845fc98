"""GPU tests of eviction from the 8-bit paged cache, and of a session that writes, attends, observes, evicts and plans, against
evict8_ref.  What is kept is exact: the order of the numbers, and codes by one rounding to nearest even."""

import numpy as np
import pytest
import torch

import evict8_ref as eref
import paged8_ref as ref
from test_gpu_paged8 import SM, bound, formats
from test_gpu_window8 import caches, check_mass, i32
from turboquant.core.rope import rope_turns
from turboquant.integration.paged_backend import PagedDecodeMetadata, TurboQuantPaged8State, TurboQuantPagedImpl
from turboquant.kernels.evict8 import allocate_mass, evict_paged8, observe_paged8
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import decode_paged8, dequantize_paged8, prefill_paged8
from turboquant.kernels.plan import new_pool, plan_step
from turboquant.kernels.rotation import apply_rope

pytestmark = pytest.mark.gpu


def tiles(dev, rng, lens, hkv, code, block, width=None, odd=False):
    """Caches of random codes and scales from 2^-12 to 2^3, mass with ties, and a table: on the CPU as evict8_ref takes them, on
    the GPU as evict_paged8 does.  odd: NaN, infinities, zero scales, NaN codes."""
    need = [-(-n // block) for n in lens]
    nb = sum(need) + 2
    fmts = formats(code, block)
    perm = rng.permutation(nb)
    bt = np.full((len(lens), width or max(need + [1])), -1, dtype=np.int32)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    got, val, exp = [], [], []
    for f in fmts:
        x = ref.codes(rng.standard_normal((nb, hkv, block, 128)) * (60 if code == "e4m3" else 40), code)
        e = rng.integers(-12, 4, (nb, hkv))
        if odd:
            if code == "e4m3":
                x[rng.random(x.shape) < 0.001] = np.nan
            e[rng.random(e.shape) < 0.1] = -999
        got.append(ref.pack(x, np.where(e > -999, 2.0 ** np.where(e > -999, e, 0), 0.0), f).to(dev))
        val.append(x)
        exp.append(e)
    mass = np.round(np.exp(rng.standard_normal((nb, hkv, block)) * 2), 1).astype(np.float32)   # many ties
    if odd:
        for x in (np.nan, np.inf, -np.inf, -0.0, 0.0, -3.5, 1e-45):
            mass[rng.random(mass.shape) < 0.05] = x
    return got, fmts, val, exp, mass, bt


def compare(dev, rng, lens, hkv, code, block, keep, recent, sinks, longer=None, cap=None, width=None, odd=False, spoil=None):
    (kc, vc), (kf, vf), val, exp, mass, bt = tiles(dev, rng, lens, hkv, code, block, width, odd)
    if spoil:
        spoil(bt)
    gm = torch.from_numpy(mass).to(dev)
    longer_than = keep if longer is None else longer
    limit = min(bt.shape[1] * block, cap if cap is not None else 1 << 30)
    first = [eref.read(c, f) for c, f in ((kc, kf), (vc, vf))]
    for (v, e), (w, x) in zip(first, zip(val, exp)):
        np.testing.assert_array_equal(v, w)
        np.testing.assert_array_equal(e, x)
    change = evict_paged8(kc, kf, vc, vf, gm, torch.from_numpy(bt).to(dev), i32(lens, dev), keep, recent=recent, sinks=sinks,
                          longer_than=longer, max_seq_len=cap)
    want = eref.evict(val, exp, mass, bt, lens, keep, recent, sinks, longer_than, limit, block, code)
    assert change.tolist() == want
    np.testing.assert_array_equal(gm.cpu().numpy(), mass)
    for c, f, v, e in ((kc, kf, val[0], exp[0]), (vc, vf, val[1], exp[1])):
        got, ge = eref.read(c, f)
        np.testing.assert_array_equal(ge, e)
        np.testing.assert_array_equal(got, v)
    return change


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [16, 48, 128])
@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (5, 0, 5), (16, 4, 2), (33, 33, 0), (100, 40, 7), (129, 0, 0),
                                               (200, 100, 100)])
def test_evict(dev, code, block, keep, recent, sinks):
    rng = np.random.default_rng(keep + block)
    lens = [0, 1, keep - 1, keep, keep + 1, keep + 15, keep + 16, 2 * keep + 3, 333, 700]
    compare(dev, rng, lens, 2, code, block, keep, recent, sinks)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [16, 64])
def test_evict_odd_contents(dev, code, block):
    """NaN, infinite, negative and zero numbers, tiles without a scale, NaN codes, bad table entries in every place."""
    rng = np.random.default_rng(block)

    def spoil(bt):
        bt[0, 1], bt[1, -1], bt[2, :], bt[3, 0] = -1, 10 ** 6, -3, 1 << 30
        bt[4, 2:] = -1

    compare(dev, rng, [400, 390, 300, 500, 450, 420], 3, code, block, 150, 30, 20, odd=True)
    compare(dev, rng, [400, 390, 300, 500, 450, 420], 3, code, block, 150, 30, 20, odd=True, spoil=spoil)
    compare(dev, rng, [400, 390, 300, 500, 450, 420], 3, code, block, 150, 0, 0, odd=True, spoil=spoil)


def test_evict_thresholds(dev):
    """longer_than, lengths behind max_seq_len or the tables, keep beyond what the tables hold, no sequence to cut."""
    rng = np.random.default_rng(9)
    compare(dev, rng, [100, 101, 160, 161, 300], 1, "e4m3", 16, 100, 10, 2, longer=160)
    compare(dev, rng, [100, 250, 300], 2, "e4m3", 16, 64, 10, 2, cap=240)
    compare(dev, rng, [100, 250, 300], 2, "int8", 16, 64, 64, 0, cap=64)
    compare(dev, rng, [100, 90], 2, "e4m3", 16, 5000, 10, 2)
    compare(dev, rng, [0, 0], 2, "e4m3", 16, 5, 1, 1, width=3)
    (kc, vc), (kf, vf), *_ , bt = tiles(dev, rng, [100, 300], 2, "e4m3", 16)
    mass = allocate_mass(kc.shape[0], 2, 16, device=dev)
    # lengths that pass the tables: the change still leads to `keep`
    out = torch.full((2,), 5, dtype=torch.int32, device=dev)
    got = evict_paged8(kc, kf, vc, vf, mass, torch.from_numpy(bt).to(dev), i32([100, 5000], dev), 150, out=out)
    assert got is out and got.tolist() == [0, 150 - 5000]


@pytest.mark.parametrize("code,block,hkv,seqs", [("e4m3", 16, 2, 110), ("int8", 48, 8, 25), ("e4m3", 64, 1, 200), ("int8", 64, 3, 63),
                                                 ("e4m3", 32, 3, 64)])
def test_evict_many_segments(dev, code, block, hkv, seqs):
    """Around the number of (sequence, KV head) pairs from which on a workgroup takes a whole one."""
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, 150, seqs)]
    compare(dev, rng, lens, hkv, code, block, 57, 11, 3, odd=True, width=11)
    lens = [int(x) for x in rng.integers(300, 420, 4)] + [0] * (seqs - 4)
    compare(dev, rng, lens, hkv, code, block, 290, 11, 3)


@pytest.mark.parametrize("n,keep", [(5000, 1700), (20000, 9001), (70001, 30000)])
def test_evict_long(dev, n, keep):
    """Rounds beyond the plan's first, against an ordering by torch; all-equal numbers keep the first tokens."""
    g = torch.Generator(device=dev).manual_seed(n)
    rng = np.random.default_rng(n)
    (kc, vc), (kf, vf), *_, bt = tiles(dev, rng, [n], 1, "int8", 16)
    for x, f in ((kc, kf), (vc, vf)):
        # (one scale everywhere: codes move as they are)
        x[..., f.code_bytes:f.code_bytes + 4] = torch.ones(x.shape[0], 1, 1, device=dev).view(torch.uint8)
    bt = torch.from_numpy(bt).to(dev)
    t = torch.arange(n, device=dev)
    blk = bt[0].long()[t // 16]
    for ties in (False, True):
        mass = torch.rand(kc.shape[0], 1, 16, generator=g, device=dev)
        if ties:
            mass = torch.floor(mass * 3)
        k, v = kc.clone(), vc.clone()
        m = mass[blk, 0, t % 16]
        body = torch.sort(m[3:n - 500], descending=True, stable=True).indices[:keep - 503] + 3
        src = torch.cat([t[:3], body.sort().values, t[n - 500:]])
        want = [dequantize_paged8(x, f)[blk[src], 0, src % 16] for x, f in ((k, kf), (v, vf))]
        evict_paged8(k, kf, v, vf, mass, bt, i32([n], dev), keep, recent=500, sinks=3)
        for x, f, w in ((k, kf, want[0]), (v, vf, want[1])):
            assert torch.equal(dequantize_paged8(x, f)[blk[:keep], 0, t[:keep] % 16], w)
        assert torch.equal(mass[blk[:keep], 0, t[:keep] % 16], m[src])


@pytest.mark.parametrize("code,block,hkv,seqs,n,keep", [
    ("e4m3", 16, 1, 200, 2600, 1500), ("int8", 48, 8, 25, 1900, 1050), ("e4m3", 64, 2, 100, 2100, 1301), ("int8", 16, 1, 193, 34000, 900)])
def test_evict_many_rounds(dev, code, block, hkv, seqs, n, keep):
    """A workgroup per (sequence, KV head), of which two sequences are cut, over 4 to 6 rounds of 256 kept rows: blocks that reach from one
    round into the next (48), scales that differ, numbers of one sequence that do not fit the plan's registers (34000)."""
    rng = np.random.default_rng(n)
    lens = [0] * seqs
    lens[3], lens[seqs - 1] = n, keep + 77
    compare(dev, rng, lens, hkv, code, block, keep, 200, 5, odd=True)


@pytest.mark.parametrize("code,block,keep", [("e4m3", 16, 9001), ("int8", 48, 4000), ("e4m3", 64, 6143)])
def test_evict_long_scales(dev, code, block, keep):
    """Few segments over many tickets, with scales that differ: a block's scale is written when no unit needs the old one."""
    rng = np.random.default_rng(keep)
    compare(dev, rng, [20000, keep + 1, 9500], 1, code, block, keep, 500, 3, odd=True)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [80, 128, 160])
def test_evict_odd_contents_of_large_blocks(dev, code, block):
    """The path through the workspace, over several kept blocks: odd contents, bad table entries, blocks of no power of two."""
    rng = np.random.default_rng(block)

    def spoil(bt):
        bt[0, 1], bt[1, -1], bt[2, :], bt[3, 0] = -1, 10 ** 6, -3, 1 << 30
        bt[4, 2:] = -1

    lens = [1400, 1390, 900, 1500, 1450, 700, 650]
    compare(dev, rng, lens, 2, code, block, 650, 90, 20, odd=True)
    compare(dev, rng, lens, 2, code, block, 650, 90, 20, odd=True, spoil=spoil)
    compare(dev, rng, lens, 2, code, block, 641, 0, 0, odd=True, spoil=spoil)


def test_evict_strided(dev):
    """K and V tiles side by side in one tensor, mass with other strides, strided lengths, a stream of its own."""
    rng = np.random.default_rng(4)
    lens = [300, 77, 180]
    (kc, vc), (kf, vf), val, exp, mass, bt = tiles(dev, rng, lens, 2, "e4m3", 16)
    both = torch.zeros(kc.shape[0], 4, 2 * kf.tile_bytes, dtype=torch.uint8, device=dev)
    both[:, ::2, :kf.tile_bytes], both[:, ::2, kf.tile_bytes:] = kc, vc
    rest = both[:, 1::2].clone()
    gm = torch.zeros(kc.shape[0], 2, 32, device=dev)
    gm[..., :16] = torch.from_numpy(mass).to(dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    wide = torch.full((3, 40), -2, dtype=torch.int32, device=dev)
    wide[:, :bt.shape[1]] = torch.from_numpy(bt).to(dev)
    with torch.cuda.stream(stream):
        change = evict_paged8(both[:, ::2, :kf.tile_bytes], kf, both[:, ::2, kf.tile_bytes:], vf, gm[..., :16], wide[:, :bt.shape[1]],
                              i32([300, 0, 77, 0, 180, 0], dev)[::2], 100, recent=20, sinks=4)
    torch.cuda.current_stream(dev).wait_stream(stream)
    assert change.tolist() == eref.evict(val, exp, mass, bt, lens, 100, 20, 4, 100, 1 << 30, 16, "e4m3")
    np.testing.assert_array_equal(gm[..., :16].cpu().numpy(), mass)
    assert not gm[..., 16:].any() and torch.equal(both[:, 1::2], rest)
    for i, f in enumerate((kf, vf)):
        got, e = eref.read(both[:, ::2, i * f.tile_bytes:(i + 1) * f.tile_bytes], f)
        np.testing.assert_array_equal(got, val[i])
        np.testing.assert_array_equal(e, exp[i])


def test_refusals(dev):
    (kc, vc), (kf, vf), _, _, mass, bt = tiles(dev, np.random.default_rng(0), [100, 50], 2, "e4m3", 16)
    good = dict(k_cache=kc, k_fmt=kf, v_cache=vc, v_fmt=vf, mass=torch.from_numpy(mass).to(dev), block_tables=torch.from_numpy(bt).to(dev),
                seq_lens=i32([100, 50], dev), keep=32)
    before = kc.clone()
    m = good["mass"]
    for kw in (dict(keep=0), dict(keep=-4), dict(recent=33), dict(sinks=20, recent=13), dict(recent=-1), dict(sinks=-1), dict(longer_than=31),
               dict(mass=m[:-1]), dict(mass=m.half()), dict(mass=m.cpu()), dict(k_fmt=vf), dict(v_cache=vc[:-1]),
               dict(k_cache=kc[..., :-16]), dict(seq_lens=i32([100], dev)), dict(block_tables=good["block_tables"][:, ::2]),
               dict(out=torch.empty(3, dtype=torch.int32, device=dev)), dict(out=torch.empty(2, dtype=torch.int64, device=dev)),
               dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev))):
        with pytest.raises(ValueError):
            evict_paged8(**{**good, **kw})
    for kw in (dict(seq_lens=good["seq_lens"].long()), dict(block_tables=good["block_tables"].long())):
        with pytest.raises(TypeError):
            evict_paged8(**{**good, **kw})
    assert torch.equal(kc, before)
    empty = evict_paged8(**{**good, "seq_lens": i32([], dev), "block_tables": good["block_tables"][:0]})
    assert empty.shape == (0,)


def test_out_apart_from_lengths(dev):
    """The heads of a sequence read its length while its change is written: a shared tensor is refused, a neighbour is not."""
    (kc, vc), (kf, vf), _, _, mass, bt = tiles(dev, np.random.default_rng(0), [100, 50], 2, "e4m3", 16)
    good = dict(k_cache=kc, k_fmt=kf, v_cache=vc, v_fmt=vf, mass=torch.from_numpy(mass).to(dev), block_tables=torch.from_numpy(bt).to(dev),
                keep=64)
    both = i32([100, 50, 7, 7, 7], dev)
    before = kc.clone()
    for at in (0, 1):
        with pytest.raises(ValueError, match="share memory"):
            evict_paged8(**good, seq_lens=both[:2], out=both[at:at + 2])
    assert torch.equal(kc, before)
    assert evict_paged8(**good, seq_lens=both[:2], out=both[2:4]).tolist() == [-36, 0]
    assert both.tolist() == [100, 50, -36, 0, 7]


class Session:
    """What a serving loop keeps, and its mirror in plain terms: per sequence and KV head the rows that are cached."""

    def __init__(self, dev, seqs, code, block, blocks=200, hkv=2, group=2):
        self.dev, self.hkv, self.hq, self.block = dev, hkv, hkv * group, block
        self.state = TurboQuantPaged8State(128, device=dev, encoding=code, block_size=block)
        self.kv = self.state.allocate_kv_cache(blocks, hkv, dev)
        self.mass = self.state.allocate_mass(blocks, hkv, dev)
        self.mass.fill_(float("nan"))                       # (recycled rows hold anything)
        self.tables = torch.full((seqs, 40), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.ring, self.pool = new_pool(blocks, dev)
        self.gone = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.turns, _ = rope_turns(device=dev)
        self.impl = TurboQuantPagedImpl(self.hq, 128, SM, hkv, self.state, mass=self.mass, observe_last=24)

    def step(self, new, q, k, v, most, decode):
        """One layer's step: new tokens per sequence, their rows; returns the outputs."""
        start = self.gone + self.lens
        plan = plan_step(self.lens, i32(new, self.dev), self.tables, self.ring, self.pool, self.block, sum(new))
        rep = torch.repeat_interleave(self.gone, i32(new, self.dev).long(), output_size=sum(new))
        q, k = apply_rope(q, k, plan.positions + rep, self.turns)
        assert torch.equal(plan.positions + rep, torch.cat([torch.arange(a, a + n, device=self.dev) for a, n in zip(start.tolist(), new)]).int())
        self.impl.do_kv_cache_update(None, k, v, self.kv, plan.slot_mapping)
        md = PagedDecodeMetadata.from_plan(plan, self.tables, 40 * self.block, num_decodes=len(new) if decode else 0, max_query_len=most)
        out = torch.empty_like(q)
        self.impl.forward(None, q, k, v, self.kv, md, out)
        self.lens = plan.seq_lens
        return out, q

    def evict(self, **kw):
        kc, vc = self.state.split_kv_cache(self.kv)
        change = self.state.evict(kc, vc, self.mass, self.tables, self.lens, **kw)
        plan = plan_step(self.lens, change, self.tables, self.ring, self.pool, self.block, 0)
        self.lens = plan.seq_lens
        self.gone = self.gone - change
        return change


@pytest.mark.parametrize("code,block", [("e4m3", 16), ("int8", 32)])
def test_session(dev, code, block):
    """Prompts, decode steps, evictions and steps after them, as a serving loop runs them: every output and every accumulated
    weight against the definitions on what the cache held, the pool whole in the end."""
    g = torch.Generator(device=dev).manual_seed(3)
    S, prompts = 3, [150, 40, 90]
    ses = Session(dev, S, code, block)

    def rows(n, heads):
        return torch.randn(n, heads, 128, generator=g, device=dev).to(torch.bfloat16)

    def expect(out, q, new, before, last):
        kc, vc = ses.state.split_kv_cache(ses.kv)
        kval, vval = (dequantize_paged8(c, f).cpu().double().numpy() for c, f in ((kc, ses.state.k_format), (vc, ses.state.v_format)))
        tables, lens, at, adds = ses.tables.cpu(), ses.lens.tolist(), 0, []
        for s, n in enumerate(new):
            want, add = eref.sequence(q[at:at + n].cpu().double().numpy(), kval, vval, tables[s], lens[s], None, 0, SM, last)
            err = np.abs(out[at:at + n].cpu().double().numpy() - want)
            assert np.all(err <= bound(np.abs(vval).max(), lens[s], out.dtype, out.dtype, want))
            adds.append(add)
            at += n
        used = torch.zeros_like(before, dtype=torch.bool)
        for s, L in enumerate(lens):
            t = torch.arange(L)
            used[tables[s][t // block].long(), :, t % block] = True
        check_mass(torch.where(used, ses.mass, 0.0), torch.where(used, before, 0.0), adds, tables, lens, new, block, 24 * ses.hq)

    before = ses.mass.clone()
    out, q = ses.step(prompts, rows(280, ses.hq), rows(280, ses.hkv), rows(280, ses.hkv), 150, False)
    expect(out, q, prompts, before, 24)
    for round_ in range(3):
        for _ in range(2):
            before = ses.mass.clone()
            out, q = ses.step([1] * S, rows(S, ses.hq), rows(S, ses.hkv), rows(S, ses.hkv), 1, True)
            expect(out, q, [1] * S, before, None)
        lens = ses.lens.tolist()
        assert not ses.mass[ses.tables[0, 0].long()].isnan().any()
        change = ses.evict(keep=60, recent=20, sinks=4, longer_than=61)
        assert change.tolist() == [60 - n if n > 61 else 0 for n in lens]
        assert ses.lens.tolist() == [60 if n > 61 else n for n in lens]
        before = ses.mass.clone()
        out, q = ses.step([30, 1, 5], rows(36, ses.hq), rows(36, ses.hkv), rows(36, ses.hkv), 30, False)
        expect(out, q, [30, 1, 5], before, 24)
    held = sum(-(-n // block) for n in ses.lens.tolist())
    assert ses.pool.tolist()[1] == 200 - held
    blocks = [ses.tables[s, i].item() for s, n in enumerate(ses.lens.tolist()) for i in range(-(-n // block))]
    assert len(set(blocks)) == held


def test_captured(dev):
    """Decode with mass and a window, observe and evict in a captured graph, replayed several times with the program's own
    work between, against eager calls on the same inputs; two graphs side by side."""
    lens, keep = [500, 61, 333], 200
    args, _ = caches(dev, lens, 2, "e4m3", 16)
    kc, kf, vc, vf, bt = args
    g = torch.Generator(device=dev).manual_seed(2)
    q = torch.randn(3, 8, 128, generator=g, device=dev).to(torch.bfloat16)
    qp = torch.randn(12, 8, 128, generator=g, device=dev).to(torch.bfloat16)
    cu, sl = i32([0, 5, 5, 12], dev), i32(lens, dev)
    mass = torch.rand(kc.shape[0], 2, 16, generator=g, device=dev)
    state = [kc, vc, mass]
    saved = [x.clone() for x in state]
    out, outp, change = torch.empty_like(q), torch.empty_like(qp), torch.empty(3, dtype=torch.int32, device=dev)
    def attend():
        decode_paged8(q, kc, kf, vc, vf, bt, sl, window=300, sinks=4, mass=mass, out=out)
        observe_paged8(qp, cu, kc, kf, bt, sl, mass, last=4)
        prefill_paged8(qp, cu, kc, kf, vc, vf, bt, sl, window=77, sinks=9, out=outp)

    def cut():
        evict_paged8(kc, kf, vc, vf, mass, bt, sl, keep, recent=50, sinks=4, out=change)

    def reset():
        for x, y in zip(state, saved):
            x.copy_(y)

    def results():
        return [x.clone() for x in (kc, vc, mass, out, outp, change)]

    want, queries = [], []
    for i in range(3):
        reset()
        q.mul_(-1.25), qp.mul_(1.5)
        queries.append((q.clone(), qp.clone()))
        attend(), cut()
        want.append(results())
    reset()
    warm = torch.cuda.Stream(dev)
    warm.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(warm):
        attend(), cut()
    torch.cuda.current_stream(dev).wait_stream(warm)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        attend()
    with torch.cuda.graph(g2):
        cut()
    for i in range(3):
        reset()
        q.copy_(queries[i][0]), qp.copy_(queries[i][1])
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for a, b in zip(results(), want[i]):
            assert torch.equal(a, b), i
        # the program's own work between replays
        decode_paged8(q, kc, kf, vc, vf, bt, sl)
