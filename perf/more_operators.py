"""Performance cases of long sessions in a bounded 8-bit paged cache.

A case's "kind":

  decode   decode_paged8 with a window: one query token per sequence sees the last `window` tokens and the first `sinks`
  prefill  prefill_paged8 with a window: the same for several new tokens per sequence
  weigh    decode_paged8 with mass: decode that adds each token's attention weights to its accumulated ones
  observe  observe_paged8: the accumulated weights of prompts, from their last queries
  evict    evict_paged8: caches cut, in place, to the tokens of largest accumulated weight

With `own` false, run() computes them in elementary torch operations.  A case holds plain values
only; lengths are drawn from the case's own "layout" number, tensors from the seed.  K and V rows
are N(0, 1) times a log-normal scale per channel with 2 % of the channels eight times larger (the
outlier channels of real keys); queries are N(0, 1).  window 0: none.

The cache: a tile per (block, KV head) of block * 128 code bytes, the tile's fp32 scale and 12 bytes
of padding.  Codes are e4m3 or int8 and stand for code * scale; the scale is a power of two.  Keys are
row-major; values have the dims of four consecutive tokens interleaved, [token / 4][dim][token % 4].
Accumulated weights: fp32 [blocks, KV heads, block], paged like the cache.
"""

import functools
import math
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "turboquant-amd_amd"))

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}


def _dev():
    return torch.device("cuda")


# ---- the cases ----------------------------------------------------------------------------

def listed():
    return [
        # one user's chat with a layer of short reach
        dict(name="window_decode_one", kind="decode", seqs=1, lo=8195, hi=8195, window=1024, sinks=4, hq=32, hkv=8,
             code="int8", block=16, dtype="f16", layout=1),
        # a server's decode step: chats of very mixed lengths, a window and the first tokens kept
        dict(name="window_decode_64", kind="decode", seqs=64, lo=300, hi=32768, window=4096, sinks=4, hq=48, hkv=8,
             code="e4m3", block=16, dtype="bf16", layout=2),
        # chunked prefill on top of long contexts, ragged
        dict(name="window_extend_6", kind="prefill", seqs=6, new_lo=37, new_hi=512, past_lo=1000, past_hi=16000,
             window=2048, sinks=64, hq=32, hkv=8, code="int8", block=32, dtype="f16", layout=3),
        # whole prompts
        dict(name="window_prompt_4x4k", kind="prefill", seqs=4, new_lo=4096, new_hi=4096, past_lo=0, past_hi=0,
             window=1024, sinks=4, hq=48, hkv=8, code="e4m3", block=16, dtype="bf16", layout=4),
        # interactive decoding of one user, weights accumulated
        dict(name="weigh_one", kind="weigh", seqs=1, lo=4099, hi=4099, window=0, sinks=0, hq=32, hkv=8, code="int8",
             block=16, dtype="bf16", layout=5),
        # a batch of chats whose caches are held to some thousand tokens
        dict(name="weigh_batch", kind="weigh", seqs=32, lo=1024, hi=8192, window=0, sinks=0, hq=32, hkv=8, code="e4m3",
             block=16, dtype="bf16", layout=6),
        # long contexts at high concurrency
        dict(name="weigh_long", kind="weigh", seqs=64, lo=32768, hi=32768, window=0, sinks=0, hq=48, hkv=8, code="e4m3",
             block=16, dtype="bf16", layout=7),
        # prompts that were just written: which of their tokens the last 32 queries look at
        dict(name="observe_last", kind="observe", seqs=4, new_lo=8000, new_hi=8192, past_lo=0, past_hi=0, last=32,
             window=0, sinks=0, hq=48, hkv=8, code="e4m3", block=16, dtype="bf16", layout=8),
        # chunks of prompts, every query counts
        dict(name="observe_chunk", kind="observe", seqs=2, new_lo=384, new_hi=512, past_lo=1000, past_hi=8000, last=512,
             window=0, sinks=0, hq=32, hkv=8, code="int8", block=16, dtype="bf16", layout=9),
        # chats held at 4096 tokens, cut every 256 new ones
        dict(name="evict_step", kind="evict", seqs=32, lo=4352, hi=4352, keep=4096, recent=1024, sinks=4, heads=8,
             code="e4m3", block=16, layout=10),
        # one long prompt cut to what its last queries look at
        dict(name="evict_prompt", kind="evict", seqs=1, lo=32768, hi=32768, keep=2048, recent=256, sinks=4, heads=8,
             code="int8", block=16, layout=11),
        # a full server's caches halved and more, lengths that are no multiples of a block
        dict(name="evict_batch", kind="evict", seqs=16, lo=3001, hi=32768, keep=8190, recent=512, sinks=64, heads=8,
             code="e4m3", block=32, layout=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8), (48, 8), (64, 8), (28, 4), (24, 4), (16, 2), (8, 8), (32, 2)]


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "weigh", "weigh", "observe", "observe", "evict", "evict"])
    hq, hkv = rng.choice(HEADS)
    case = dict(kind=kind, code=rng.choice(["e4m3", "e4m3", "int8"]), block=rng.choice([16, 16, 16, 32, 64]),
                layout=rng.randrange(1 << 20))
    if kind == "evict":
        hi = _log(rng, 100, 32768)
        keep = min(_log(rng, 32, 8192), hi - 1)
        sinks = min(rng.choice([0, 4, 64]), keep // 4)
        return dict(case, seqs=_log(rng, 1, min(32, max(1, 400000 // hi))), lo=max(keep // 2, hi // rng.choice([1, 2, 8])),
                    hi=hi, keep=keep, recent=keep // rng.choice([2, 4, 16]), sinks=sinks, heads=hkv)
    window = rng.choice([0, _log(rng, 1, 8192)]) if kind in ("weigh", "observe") else _log(rng, 1, 8192)
    case.update(window=window, sinks=rng.choice([0, 1, 4, 37, 128]) if window else 0, hq=hq, hkv=hkv,
                dtype=rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"]))
    if kind in ("decode", "weigh"):
        hi = _log(rng, 64, 32768)
        return dict(case, seqs=_log(rng, 1, 48), lo=max(1, hi // rng.choice([1, 1, 8])), hi=hi)
    seqs = _log(rng, 1, 8)
    past = rng.choice([0, 0, 2000, 8000])
    hi = _log(rng, 16, 4096 if seqs <= 2 and not past else 6144 // max(seqs, 3))
    case.update(seqs=seqs, new_lo=min(hi, _log(rng, 1, 64)), new_hi=hi, past_lo=0, past_hi=past)
    return dict(case, last=rng.choice([1, 16, 32, 64, 4096])) if kind == "observe" else case


# ---- lengths and rows: shared by prepare, work and exact ------------------------------------

def _between(rng, lo, hi):
    """Log-uniform over wide ranges, uniform over narrow ones."""
    if lo >= hi:
        return hi
    return _log(rng, lo, hi) if hi > 10 * max(lo, 1) and lo > 0 else rng.randint(lo, hi)


def _lens(case):
    """(lengths before, new tokens) of the case's sequences, on the host."""
    rng = random.Random(case["layout"])
    if case["kind"] in ("decode", "weigh", "evict"):
        return [_between(rng, case["lo"], case["hi"]) - 1 for _ in range(case["seqs"])], [1] * case["seqs"]
    new = [_between(rng, case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    return [_between(rng, case["past_lo"], case["past_hi"]) for _ in new], new


def _gen(seed, part):
    return torch.Generator(device=_dev()).manual_seed((int(seed) * 1000003 + part) % (1 << 62))


def _randn(shape, seed, part):
    return torch.randn(shape, generator=_gen(seed, part), device=_dev())


def _scales(seed, heads):
    """Per-channel scales of K and of V."""
    out = []
    for part in (999983, 999959):
        s = torch.exp(_randn((heads, D), seed, part) * 0.5)
        out.append(torch.where(torch.rand(heads, D, generator=_gen(seed, part + 1), device=_dev()) < 0.02, s * 8, s))
    return out


def _tables(total, block, seed, spare=8):
    """Block table [S, max blocks] over a random permutation of the pool, and the pool's size."""
    blocks = [-(-n // block) for n in total]
    nb = sum(blocks) + spare
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
    bt = torch.full((len(total), max(max(blocks), 1)), -1, dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        bt[s, :b] = perm[at:at + b]
        at += b
    return bt, nb


# ---- the 8-bit tiles, in plain operations ------------------------------------------------------

def _exponent(top, code):
    """The smallest e >= -126 with top <= TOP * 2^e, as int32."""
    m, e = torch.frexp(top)                                # top = m 2^e, m in [0.5, 1)
    lim, le = math.frexp(TOP[code])
    return torch.where(top > 0, e - le + (m > lim).to(torch.int32), torch.full_like(e, -126)).clamp(min=-126)


def _encode(y, code):
    """Codes of scaled fp32 values, as bytes."""
    if code == "e4m3":
        return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return y.round().clamp(-127.0, 127.0).to(torch.int8).view(torch.uint8)


def _interleave(b):
    """Value bytes [..., block, 128] row-major -> the values layout, flat."""
    return b.reshape(*b.shape[:-2], -1, 4, D).transpose(-1, -2).reshape(*b.shape[:-2], -1)


def _rows(flat, values):
    """Code bytes of tiles [..., block * 128] -> [..., block, 128]."""
    if values:
        return flat.reshape(*flat.shape[:-1], -1, D, 4).transpose(-1, -2).reshape(*flat.shape[:-1], -1, D)
    return flat.reshape(*flat.shape[:-1], -1, D)


def _decode(b, code):
    return b.contiguous().view(CODE[code]).to(torch.float32)


def _parts(cache, block, code):
    """What a cache holds: its codes in their type and its scales (views)."""
    n = block * D
    return cache[..., :n].view(CODE[code]), cache[..., n:n + 4].view(torch.float32)


def _fill(caches, s, n, bt, seed, case, heads, spread):
    """Fills the blocks of sequence s; a token's rows have a log-normal size of deviation `spread`."""
    block, sc = case["block"], _scales(seed, heads)
    nb = -(-n // block)
    at = bt[s, :nb].long().to(_dev())
    for i, cache in enumerate(caches):
        x = (_randn((nb, block, heads, D), seed, 2 * s + i) * sc[i]).transpose(1, 2)
        if spread:
            x = x * torch.exp(spread * _randn((nb, heads, block, 1), seed, 500000 + 2 * s + i))
        scale = torch.ldexp(torch.ones(nb, heads, device=_dev()), _exponent(x.abs().amax((2, 3)), case["code"]))
        codes = _encode(x / scale[..., None, None], case["code"])
        tail = torch.zeros(nb, heads, 16, dtype=torch.uint8, device=_dev())
        tail[..., :4] = scale.view(torch.uint8).reshape(nb, heads, 4)
        cache[at] = torch.cat([_interleave(codes) if i else codes.flatten(2), tail], -1)


# ---- prepare ---------------------------------------------------------------------------------

def prepare(case, seed):
    past, new = _lens(case)
    total = [p + n for p, n in zip(past, new)]
    block, evict = case["block"], case["kind"] == "evict"
    heads = case["heads"] if evict else case["hkv"]
    bt, nb = _tables(total, block, seed)
    kc, vc = (torch.zeros(nb, heads, block * D + 16, dtype=torch.uint8, device=_dev()) for _ in range(2))
    for s, n in enumerate(total):
        _fill((kc, vc), s, n, bt, seed, case, heads, 0.5 if evict else 0.0)
    st = dict(case=case, kc=kc, vc=vc, bt=bt.to(_dev()), longest=max(total),
              lens=torch.tensor(total, dtype=torch.int32, device=_dev()))
    if case["kind"] in ("weigh", "observe", "evict"):
        # weights of earlier steps: a few tokens have most, some none
        x = torch.exp(2.0 * _randn((nb, heads, block), seed, 900001) - 4.0)
        st["mass"] = torch.where(torch.rand(x.shape, generator=_gen(seed, 900002), device=_dev()) < 0.1, torch.zeros_like(x), x)
    if not evict:
        st["q"] = _randn((sum(new), case["hq"], D), seed, 900003).to(DTYPES[case["dtype"]])
        st["out"] = torch.empty_like(st["q"])
    if case["kind"] in ("prefill", "observe"):
        at = [0]
        for n in new:
            at.append(at[-1] + n)
        st.update(cu=torch.tensor(at, dtype=torch.int32, device=_dev()), most=max(new))
    return st


# ---- run ---------------------------------------------------------------------------------------

def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


@functools.lru_cache(maxsize=None)
def _formats(code, block):
    from turboquant.kernels.paged8 import Paged8Format
    return Paged8Format.for_keys(code, block), Paged8Format.for_values(code, block)


def _reach(case):
    return dict(window=case["window"], sinks=case["sinks"]) if case["window"] else {}


def _own_decode(st):
    from turboquant.kernels.paged8 import decode_paged8
    kf, vf = _formats(st["case"]["code"], st["case"]["block"])
    return decode_paged8(st["q"], st["kc"], kf, st["vc"], vf, st["bt"], st["lens"], max_seq_len=st["longest"],
                         out=st["out"], **_reach(st["case"]))


def _own_weigh(st):
    from turboquant.kernels.paged8 import decode_paged8
    kf, vf = _formats(st["case"]["code"], st["case"]["block"])
    out = decode_paged8(st["q"], st["kc"], kf, st["vc"], vf, st["bt"], st["lens"], max_seq_len=st["longest"],
                        out=st["out"], mass=st["mass"], **_reach(st["case"]))
    return dict(out=out, mass=st["mass"])


def _own_prefill(st):
    from turboquant.kernels.paged8 import prefill_paged8
    kf, vf = _formats(st["case"]["code"], st["case"]["block"])
    return prefill_paged8(st["q"], st["cu"], st["kc"], kf, st["vc"], vf, st["bt"], st["lens"], max_q_len=st["most"],
                          out=st["out"], **_reach(st["case"]))


def _own_observe(st):
    from turboquant.kernels.evict8 import observe_paged8
    kf, _ = _formats(st["case"]["code"], st["case"]["block"])
    return observe_paged8(st["q"], st["cu"], st["kc"], kf, st["bt"], st["lens"], st["mass"], last=st["case"]["last"],
                          max_q_len=st["most"], max_seq_len=st["longest"], **_reach(st["case"]))


def _own_evict(st):
    from turboquant.kernels.evict8 import evict_paged8
    c = st["case"]
    kf, vf = _formats(c["code"], c["block"])
    # (between two evictions a program's decode steps change the weights: each pass takes them as they were)
    mass = st["mass"].clone()
    change = evict_paged8(st["kc"], kf, st["vc"], vf, mass, st["bt"], st["lens"], c["keep"], recent=c["recent"],
                          sinks=c["sinks"], max_seq_len=st["longest"])
    return dict(change=change, mass=mass, k=_parts(st["kc"], c["block"], c["code"]), v=_parts(st["vc"], c["block"], c["code"]))


def _gather(cache, bt, block, code, values):
    """fp32 rows [S, Hkv, blocks * block, 128] of block tables."""
    t = cache[bt.clamp(min=0).long()].transpose(1, 2)
    n = block * D
    x = _decode(_rows(t[..., :n], values), code)
    return (x * t[..., n:n + 4].contiguous().view(torch.float32)[..., None]).flatten(2, 3)


def _visible(st):
    """The table columns that one query token per sequence needs: blocks [S, C], their tokens' positions and which of
    them it sees [S, C * block]."""
    c = st["case"]
    block, bt, lens = c["block"], st["bt"], st["lens"].long()
    width = bt.shape[1]
    lo = (lens - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(lens)
    first = min(-(-c["sinks"] // block), width)
    count = min(-(-c["window"] // block) + 1, width) if c["window"] else width
    col = torch.cat([torch.arange(first, device=bt.device).expand(len(lens), -1),
                     (lo // block).clamp(min=first)[:, None] + torch.arange(count, device=bt.device)], 1)
    pos = (col[..., None] * block + torch.arange(block, device=bt.device)).flatten(1)
    seen = (pos < lens[:, None]) & ((pos >= lo[:, None]) | (pos < c["sinks"]))
    return bt.gather(1, col.clamp(max=width - 1)), pos, seen


def _step(st):
    """Decode: the output, the weights [S, Hkv, G, tokens] and what _visible gives."""
    c = st["case"]
    bt, pos, seen = _visible(st)
    k = _gather(st["kc"], bt, c["block"], c["code"], False)
    v = _gather(st["vc"], bt, c["block"], c["code"], True)
    S, H = k.shape[:2]
    q = st["q"].float().reshape(S, H, -1, D)
    p = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    p = torch.softmax(p.masked_fill(~seen[:, None, None], -math.inf), -1)
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    return torch.matmul(p, v).reshape(st["q"].shape).to(st["q"].dtype), p, bt, pos, seen


def _plain_decode(st):
    return _step(st)[0]


def _accumulate(st, weights, bt, pos, seen, new):
    """mass += weights [S, Hkv, tokens] where seen; the tokens from position L - new[s] on start from 0."""
    block = st["case"]["block"]
    S, H = weights.shape[:2]
    old = st["mass"][bt.clamp(min=0).long()].transpose(1, 2).flatten(2)
    fresh = pos >= (st["lens"].long() - new)[:, None]
    got = torch.where(fresh[:, None], torch.zeros_like(old), old) + weights.masked_fill(~seen[:, None], 0.0)
    used = (pos < st["lens"][:, None]).view(S, -1, block)
    tok = used[:, None] & torch.ones(1, H, 1, 1, dtype=torch.bool, device=pos.device)
    got = torch.where(tok, got.view(S, H, -1, block), old.view(S, H, -1, block)).transpose(1, 2)
    real = used.any(-1)
    st["mass"][bt[real].long()] = got[real]
    return st["mass"]


def _plain_weigh(st):
    out, p, bt, pos, seen = _step(st)
    return dict(out=out, mass=_accumulate(st, p.sum(2), bt, pos, seen, 1))


def _chunk(st, last):
    """Several new tokens per sequence, the last `last` of each as queries: weights [S, Hkv, G, n, L], of rows padded
    at their front, and the (sequence, row) of every query."""
    c = st["case"]
    k = _gather(st["kc"], st["bt"], c["block"], c["code"], False)
    S, H, L, _ = k.shape
    cu, lens, q = st["cu"].long(), st["lens"].long(), st["q"].float()
    T, hq, _ = q.shape
    G, n = hq // H, min(st["most"], last)
    t = torch.arange(T, device=q.device)
    s = torch.searchsorted(cu[1:], t, right=True)
    i = n - (cu[s + 1] - t)                       # row in the padded queries; below 0: no query
    pad = torch.zeros(S, n, H, G, D, device=q.device)
    if n < st["most"]:
        t = t[i >= 0]
        s, i = s[t], i[t]
    pad[s, i] = q[t].reshape(-1, H, G, D)
    pad = pad.permute(0, 2, 3, 1, 4).reshape(S, H, G * n, D)
    p = torch.matmul(pad, k.transpose(-1, -2)).div_(math.sqrt(D)).view(S, H, G, n, L)
    at = lens[:, None] - n + torch.arange(n, device=q.device)          # the rows' positions
    key = torch.arange(L, device=q.device)
    hide = key > at[..., None]
    if c["window"]:
        hide |= (key <= (at - c["window"])[..., None]) & (key >= c["sinks"])
    rows = torch.arange(n, device=q.device) >= n - (cu[1:] - cu[:-1])[:, None]
    p = torch.softmax(p.masked_fill_(hide[:, None, None], -math.inf), -1)
    return p.masked_fill_(~rows[:, None, None, :, None], 0.0), s, i


def _plain_prefill(st):
    c = st["case"]
    p, s, i = _chunk(st, st["most"])
    v = _gather(st["vc"], st["bt"], c["block"], c["code"], True)
    S, H, L, _ = v.shape
    v = v.masked_fill((torch.arange(L, device=v.device) >= st["lens"][:, None])[:, None, :, None], 0.0)
    G, n = p.shape[2:4]
    o = torch.matmul(p.view(S, H, G * n, L), v).view(S, H, G, n, D)
    return o.permute(0, 3, 1, 2, 4)[s, i].reshape(st["q"].shape).to(st["q"].dtype)


def _plain_observe(st):
    p, _, _ = _chunk(st, st["case"]["last"])
    L = p.shape[-1]
    pos = torch.arange(L, device=p.device).expand(p.shape[0], -1)
    cu = st["cu"].long()
    return _accumulate(st, p.sum((2, 3)), st["bt"], pos, pos < st["lens"][:, None], cu[1:] - cu[:-1])


def _plain_evict(st):
    c = st["case"]
    block, code, keep, n = c["block"], c["code"], c["keep"], c["block"] * D
    bt, lens, mass = st["bt"], st["lens"].long(), st["mass"].clone()
    S, H = bt.shape[0], mass.shape[1]
    blocks = bt.clamp(min=0).long()
    cut = lens > keep
    m = mass[blocks].transpose(1, 2).flatten(2)                                              # [S, H, L]
    t = torch.arange(m.shape[2], device=m.device)
    always = (t < c["sinks"]) | (t >= (lens - c["recent"])[:, None])
    key = m.masked_fill(always[:, None], math.inf).masked_fill((t >= lens[:, None])[:, None], -math.inf)
    src = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    to = -(-keep // block)                                                                   # blocks that are kept
    some = src.shape[2]
    src = torch.nn.functional.pad(src, (0, to * block - some))
    held = torch.arange(to * block, device=m.device) < min(keep, some)
    rows, cols = torch.nonzero(cut[:, None] & (torch.arange(to, device=m.device) < bt.shape[1]), as_tuple=True)
    dst = blocks[rows, cols]

    def put(new, old):
        """[S, H, to, block, ...] kept rows, other rows as they are, for the blocks of the sequences that are cut."""
        h = held.view(to, 1, block, *[1] * (new.dim() - 4))
        new = new.transpose(1, 2)[rows, cols]
        return torch.where(h[cols], new, old)

    moved = []
    for i, cache in enumerate((st["kc"], st["vc"])):
        tiles = cache[blocks].transpose(1, 2)                                                # [S, H, blocks, bytes]
        x = _rows(tiles[..., :n], i == 1).flatten(2, 3)
        x = _decode(x.gather(2, src[..., None].expand(-1, -1, -1, D)), code).view(S, H, to, block, D)
        sc = tiles[..., n:n + 4].contiguous().view(torch.float32)[..., 0].gather(2, src // block).view(S, H, to, block)
        sc = sc.masked_fill(~held.view(to, block), 0.0)
        after = sc.amax(-1)
        x = x * torch.where(after > 0, 1.0 / after, torch.zeros_like(after))[..., None, None] * sc[..., None]
        codes = put(_encode(x, code).view(S, H, to, block, D), _rows(cache[dst][..., :n], i == 1))
        moved.append((_interleave(codes) if i else codes.flatten(2), after.transpose(1, 2)[rows, cols]))
    for cache, (codes, after) in zip((st["kc"], st["vc"]), moved):
        cache[dst, :, :n] = codes
        cache[dst, :, n:n + 4] = after.contiguous().view(torch.uint8).reshape(*after.shape, 4)
    mass[dst] = put(m.gather(2, src).view(S, H, to, block), mass[dst])
    change = torch.where(cut, keep - lens, torch.zeros_like(lens)).to(torch.int32)
    return dict(change=change, mass=mass, k=_parts(st["kc"], block, code), v=_parts(st["vc"], block, code))


# ---- work ---------------------------------------------------------------------------------------

def _pairs(case, p, n):
    """(query, key) pairs of n queries at positions p .. p + n - 1, of those the keys that any of them sees."""
    W, sinks = case["window"], case["sinks"]
    if not W:
        return n * p + n * (n + 1) // 2, p + n
    count = sum(min(i + 1, W) + min(sinks, max(i + 1 - W, 0)) for i in range(p, p + n))
    lo = max(p + 1 - W, 0)
    return count, p + n - lo + min(sinks, lo)


def work(case):
    past, new = _lens(case)
    block = case["block"]
    if case["kind"] == "evict":
        total = [p + 1 for p in past if p + 1 > case["keep"]]
        kept = len(total) * case["keep"] * case["heads"]
        return dict(bytes=sum(total) * case["heads"] * 4 + kept * (4 * D + 4) + sum(-(-t // block) for t in total) * 4,
                    flops=4 * sum(total) * case["heads"])
    counts = []
    for p, n in zip(past, new):
        rows = min(n, case["last"]) if case["kind"] == "observe" else n
        counts.append((rows, *_pairs(case, p + n - rows, rows)))
    rows, pairs, keys = (sum(x) for x in zip(*counts))
    each = {"decode": 2 * D, "prefill": 2 * D, "weigh": 2 * D + 8, "observe": D + 8}[case["kind"]]
    data = keys * case["hkv"] * each + keys // block * (8 * case["hkv"] + 4)
    data += (1 if case["kind"] == "observe" else 2) * rows * case["hq"] * D * SIZE[case["dtype"]]
    return dict(bytes=data, flops=(2 if case["kind"] == "observe" else 4) * D * pairs * case["hq"])


# ---- exact --------------------------------------------------------------------------------------

def _sequence(case, cache, blocks, count, values):
    """The first `count` rows of a sequence: [Hkv, count, 128] in 64 bits."""
    tiles = cache[blocks]
    n = case["block"] * D
    scale = tiles[..., n:n + 4].contiguous().view(torch.float32).double()
    x = tiles[..., :n].contiguous().view(CODE[case["code"]]).double() * scale
    x = x.view(*x.shape[:2], -1, D, 4).transpose(-1, -2) if values else x.view(*x.shape[:2], -1, 4, D)
    return x.flatten(2, 3).transpose(0, 1).flatten(1, 2)[:, :count].contiguous()


def exact(case, seed):
    past, new = _lens(case)
    kind = case["kind"]
    if kind == "evict":
        return _exact_evict(case, prepare(case, seed))
    seen = [min(n, case["last"]) if kind == "observe" else n for n in new]
    if sum(n * (p + m) for p, m, n in zip(past, new, seen)) * case["hq"] > 4e9:
        return None
    st = prepare(case, seed)
    out = torch.empty_like(st["q"], dtype=torch.float64)
    mass = st["mass"].double() if "mass" in st else None
    G, block, at = case["hq"] // case["hkv"], case["block"], 0
    for s, (p, n, rows) in enumerate(zip(past, new, seen)):
        L = p + n
        blocks = st["bt"][s, :-(-L // block)].long()
        k = _sequence(case, st["kc"], blocks, L, False)
        v = _sequence(case, st["vc"], blocks, L, True) if kind != "observe" else None
        q = st["q"][at + n - rows:at + n].double()
        i = torch.arange(L - rows, L, device=q.device)[:, None]
        j = torch.arange(L, device=q.device)[None]
        see = (j <= i) & ((j > i - case["window"]) | (j < case["sinks"])) if case["window"] else j <= i
        weight = torch.zeros(case["hkv"], L, dtype=torch.float64, device=q.device)
        for h in range(case["hq"]):
            sc = torch.where(see, (q[:, h] @ k[h // G].T) * D ** -0.5, torch.full((), -math.inf, dtype=torch.float64, device=q.device))
            w = torch.exp(sc - sc.amax(1, keepdim=True))
            w = w / w.sum(1, keepdim=True)
            weight[h // G] += w.sum(0)
            if v is not None:
                out[at:at + n, h] = w @ v[h // G]
        at += n
        if mass is not None:
            t = torch.arange(L, device=q.device)
            old = mass[blocks[t // block], :, t % block]
            old[p:] = 0.0
            mass[blocks[t // block], :, t % block] = old + weight.T
    return {"decode": out, "prefill": out, "weigh": dict(out=out, mass=mass), "observe": mass}[kind]


def _grid(y, code):
    """The nearest code values (ties to even) of 64-bit numbers, as numbers."""
    if code == "int8":
        return torch.round(y).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_evict(case, st):
    """Sequence by sequence and head by head from the definition."""
    block, code, keep, sinks, recent = (case[x] for x in ("block", "code", "keep", "sinks", "recent"))
    mass, change = st["mass"].double(), []
    val, scale = [], []
    for i, cache in enumerate((st["kc"], st["vc"])):
        c, s = _parts(cache, block, code)
        val.append(_rows(c.double(), i == 1))                                                # [N, H, block, 128]
        scale.append(s[..., 0].double().clone())
    old = [(v.clone(), s.clone()) for v, s in zip(val, scale)]
    before = mass.clone()
    for s, L in enumerate(st["lens"].tolist()):
        change.append(keep - L if L > keep else 0)
        if L <= keep:
            continue
        bt = st["bt"][s].long()
        t = torch.arange(L, device=mass.device)
        for h in range(mass.shape[1]):
            m = before[bt[t // block], h, t % block]
            body = m[sinks:L - recent].cpu().numpy()
            heavy = sorted((-body).argsort(kind="stable")[:keep - sinks - recent] + sinks)
            src = torch.tensor(list(range(sinks)) + [int(x) for x in heavy] + list(range(L - recent, L)), device=mass.device)
            to, to_row = bt[t[:keep] // block], t[:keep] % block
            frm, frm_row = bt[src // block], src % block
            mass[to, h, to_row] = m[src]
            for i in range(2):
                v0, s0 = old[i]
                mine = s0[frm, h]
                top = torch.nn.functional.pad(mine, (0, -keep % block)).view(-1, block).amax(1)
                scale[i][bt[:len(top)], h] = top
                val[i][to, h, to_row] = _grid(v0[frm, h, frm_row] * (mine / top[t[:keep] // block])[:, None], code)
    parts = []
    for i in range(2):
        flat = val[i].view(*val[i].shape[:2], -1, 4, D).transpose(-1, -2) if i else val[i]
        parts.append((None if code == "int8" else flat.reshape(*val[i].shape[:2], -1), scale[i][..., None]))
    return dict(change=torch.tensor(change, dtype=torch.int32, device=mass.device), mass=mass, k=parts[0], v=parts[1])
