"""GPU tests of plan_step against a step-by-step implementation, and of the operators together: a serving loop of
plan_step, apply_rope, cache writes and attention."""

import math
import random

import numpy as np
import pytest
import torch

import paged8_ref as ref
from turboquant.core.rope import rope_turns
from turboquant.integration.paged_backend import (PagedDecodeMetadata, TurboQuantPaged8State, TurboQuantPagedConfig,
                                                  TurboQuantPagedImpl, TurboQuantPagedState)
from turboquant.kernels.paged8 import decode_paged8, prefill_paged8
from turboquant.kernels.plan import new_pool, plan_step
from turboquant.kernels.rotation import apply_rope

pytestmark = pytest.mark.gpu


def plain(past, new, tables, ring, pool, bs, T):
    """The step on Python lists; returns everything as the call leaves it."""
    N, width = len(ring), len(tables[0]) if tables else 0
    first, count = pool
    tables, ring = [list(r) for r in tables], list(ring)
    lens, start, pos, slots, given_back = [], [0], [], [], []
    asked = taken = 0
    for s, (p, n) in enumerate(zip(past, new)):
        p = max(p, 0)
        total = max(p + n, 0)
        have, want = -(-p // bs), -(-total // bs)
        fits = want <= width
        need = max(0, want - have) if fits else 0
        asked += need
        given = fits and (need == 0 or asked <= count)
        if given:
            for j in range(need):
                tables[s][have + j] = ring[(first + taken + j) % N]
            taken += need
        if want < have:
            given_back += [tables[s][j] for j in range(want, min(have, width))]
        lens.append(total if given else p)
        start.append(start[-1] + max(n, 0))
        for i in range(max(n, 0)):
            pos.append(p + i)
            slots.append(tables[s][(p + i) // bs] * bs + (p + i) % bs if given else -1)
    for j, b in enumerate(given_back):
        ring[(first + count + j) % N] = b
    pos, slots = (pos + [0] * T)[:T], (slots + [-1] * T)[:T]
    return tables, ring, [(first + taken) % N, min(count - taken + len(given_back), N)], start, lens, pos, slots


def both(dev, past, new, tables, ring, pool, bs, T, alias=False):
    t = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (past, new, tables, ring, pool)]
    if not tables:
        t[2] = torch.zeros(0, 4, dtype=torch.int32, device=dev)
    want = plain(past, new, tables, ring, pool, bs, T)
    out = None
    after = torch.full((2,), -9, dtype=torch.int32, device=dev)
    if alias:                                     # in place: the lengths and the pool
        out = plan_step(t[0], t[1], t[2].clone(), t[3].clone(), t[4].clone(), bs, T)
        out.seq_lens = t[0]
    p = plan_step(t[0], t[1], t[2], t[3], t[4], bs, T, pool_out=None if alias else after, out=out)
    got = [t[2].tolist(), t[3].tolist(), p.pool.tolist(), p.query_start_loc.tolist(), p.seq_lens.tolist(), p.positions.tolist(),
           p.slot_mapping.tolist()]
    for name, a, b in zip(("tables", "ring", "pool", "starts", "lens", "positions", "slots"), got, want):
        assert a == b, name
    if not alias:
        assert t[4].tolist() == list(pool)
    return want


def scene(rng, S, width, bs, N, most_new, T=None, ended=0.2):
    """Random requests whose blocks and the free ones make up a pool of N."""
    ids = list(range(N))
    rng.shuffle(ids)
    past, tables = [], []
    for _ in range(S):
        b = rng.randint(0, min(width, 6))
        if b > len(ids):
            b = 0
        past.append(max(0, b * bs - rng.randint(0, bs - 1)) if b else 0)
        b = -(-past[-1] // bs)
        tables.append([ids.pop() for _ in range(b)] + [-1] * (width - b))
    new = [-rng.randint(0, p) if rng.random() < ended else rng.randint(0, most_new) for p in past]
    first = rng.randrange(N)
    ring = [-7] * N
    for i, b in enumerate(ids):
        ring[(first + i) % N] = b
    total = sum(max(n, 0) for n in new)
    return past, new, tables, ring, [first, len(ids)], bs, total + 3 if T is None else T


@pytest.mark.parametrize("S,N,most,bs", [(1, 8, 5, 16), (7, 200, 40, 16), (64, 1000, 1, 16), (513, 4000, 9, 32), (600, 30000, 100, 16),
                                         (20, 4000, 500, 64), (2, 3, 100, 16), (40, 130, 60, 16), (1030, 3500, 3, 48)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan_step(dev, S, N, most, bs, alias):
    """Sizes on both sides of one workgroup, rings that wrap and that run out, narrow tables, requests that end."""
    for seed in range(3):
        rng = random.Random(seed * 7919 + S)
        both(dev, *scene(rng, S, rng.choice([3, 7, 40]), bs, N, most), alias=alias)


def test_plan_step_edges(dev):
    """No requests, no tokens, too small a token array, an empty ring, lengths at block borders."""
    assert both(dev, [], [], [], [0, 1, 2], [1, 3], 16, 4)[5] == [0] * 4
    both(dev, [5, 16, 17], [0, 0, 0], [[0, 9], [1, 9], [2, 3]], [4, 5, 6, 7, 0, 0, 0, 0], [0, 4], 16, 0)
    both(dev, [0, 0], [40, 16], [[-1] * 3, [-1] * 3], [4, 5, 6, 7], [3, 4], 16, 20)       # fewer places than tokens
    both(dev, [16, 15, 0], [1, 1, 1], [[0, -1], [1, -1], [-1, -1]], [9, 8, 7, 6], [2, 0], 16, 3)
    both(dev, [16, 15, 0], [1, 1, 1], [[0, -1], [1, -1], [-1, -1]], [9, 8, 7, 6], [3, 1], 16, 3)
    both(dev, [48, 32, 31], [-48, -1, -16], [[0, 1, 2], [3, 4, -1], [5, 6, -1]], [-1] * 8, [6, 0], 16, 2)
    both(dev, [100], [-200], [[0, 1, 2, 3, 4, 5, 6]], [-1] * 8, [0, 0], 16, 1)


def test_plan_step_many_steps(dev):
    """A pool over 60 steps of requests that grow, roll back, end and begin: no block is held twice or lost, and every
    table matches the step-by-step implementation."""
    rng = random.Random(5)
    S, N, bs, width = 12, 50, 16, 9
    ring, pool = new_pool(N, dev)
    tables = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(S, dtype=torch.int32, device=dev)
    host = ([0] * S, [[-1] * width for _ in range(S)], list(range(N)), [0, N])
    for _ in range(60):
        new = [rng.choice([1, 1, rng.randint(0, 60), -rng.randint(0, n) if n else 0, -n]) for n in host[0]]
        T = 400
        p = plan_step(lens, torch.tensor(new, dtype=torch.int32, device=dev), tables, ring, pool, bs, T)
        t, r, po, start, ln, pos, slots = plain(host[0], new, host[1], host[2], host[3], bs, T)
        assert p.slot_mapping.tolist() == slots and p.positions.tolist() == pos and p.seq_lens.tolist() == ln
        assert tables.tolist() == t and ring.tolist() == r and pool.tolist() == po
        lens, host = p.seq_lens, (ln, t, r, po)
        held = [b for s in range(S) for b in t[s][:-(-ln[s] // bs)]]
        free = [r[(po[0] + i) % N] for i in range(po[1])]
        assert sorted(held + free) == list(range(N))


def test_plan_step_graph(dev):
    """A captured step, replayed with eager work between: lengths and pool move on in place."""
    S, N, bs = 4, 64, 16
    ring, pool = new_pool(N, dev)
    tables = torch.full((S, 12), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(S, dtype=torch.int32, device=dev)
    new = torch.tensor([5, 1, 0, 40], dtype=torch.int32, device=dev)
    plan = plan_step(lens, new, tables.clone(), ring.clone(), pool.clone(), bs, 64)
    plan.seq_lens = lens
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan_step(lens, new, tables, ring, pool, bs, 64, out=plan)
    host = ([0] * S, [[-1] * 12 for _ in range(S)], list(range(N)), [0, N])
    for it in range(5):
        n = [[5, 1, 0, 40], [1, 1, 1, 1], [20, -2, 3, -41], [1, 1, 1, 1], [-26, 9, 1, 0]][it]
        new.copy_(torch.tensor(n, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        t, r, po, start, ln, pos, slots = plain(*host[:1], n, *host[1:], bs, 64)
        assert (lens.tolist(), tables.tolist(), ring.tolist(), pool.tolist()) == (ln, t, r, po)
        assert plan.slot_mapping.tolist() == slots and plan.query_start_loc.tolist() == start
        host = (ln, t, r, po)


def test_plan_step_refusals(dev):
    from turboquant._lib import TurboQuantError
    i = lambda *x: torch.zeros(*x, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(past_lens=i(2), new_lens=i(2), block_tables=i(2, 3), ring=i(4), pool=i(2), block_size=16, num_tokens=4)
    plan_step(**ok)
    for kw in (dict(new_lens=i(3)), dict(block_tables=i(3, 3)), dict(block_tables=i(2)), dict(ring=i(0)), dict(pool=i(3)),
               dict(pool_out=i(1)), dict(num_tokens=-1), dict(past_lens=i(2).cpu()), dict(block_tables=i(3, 2).t())):
        with pytest.raises(ValueError):
            plan_step(**{**ok, **kw})
    for kw in (dict(past_lens=i(2).long()), dict(ring=i(4).float())):
        with pytest.raises(TypeError):
            plan_step(**{**ok, **kw})
    for kw in (dict(block_size=0), dict(block_size=8)):
        with pytest.raises(TurboQuantError):
            plan_step(**{**ok, **kw})
    with pytest.raises(ValueError):
        plan_step(**ok, out=plan_step(**{**ok, "num_tokens": 5}))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_serving_loop(dev, code):
    """plan_step -> apply_rope -> do_kv_cache_update -> forward of an 8-bit layer over steps that mix prompts, single
    tokens and rollbacks, against attention in 64 bits over the cache's values, which are followed row by row."""
    Hq, Hkv, bs, N, S = 8, 2, 16, 40, 3
    state = TurboQuantPagedConfig(128, num_layers=8, protected_bits=8, protected_encoding=code).get_state(0, device=dev)
    assert isinstance(state, TurboQuantPaged8State)
    impl = TurboQuantPagedImpl(Hq, 128, 1 / math.sqrt(128), Hkv, state)
    assert impl.get_kv_cache_shape(N, bs, Hkv, 128, k_bits=8) == state.kv_cache_shape(N, Hkv)
    cache = state.allocate_kv_cache(N, Hkv)
    turns, mag = rope_turns(96, device=dev)
    ring, pool = new_pool(N, dev)
    tables = torch.full((S, 12), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(S, dtype=torch.int32, device=dev)
    kref, vref = ref.Cache(N, Hkv, bs, code), ref.Cache(N, Hkv, bs, code)
    g = torch.Generator().manual_seed(9)
    for new, decodes in (([5, 40, 17], 0), ([1, 1, 1], None), ([1, 1, 30], 2), ([-2, -3, -47], None), ([1, 1, 1], None),
                         ([1, 70, 3], 1)):
        T = sum(max(n, 0) for n in new)
        plan = plan_step(lens, torch.tensor(new, dtype=torch.int32, device=dev), tables, ring, pool, bs, T + 2)
        lens = plan.seq_lens
        if not T:
            continue
        q, k, v = (torch.randn(T + 2, h, 128, generator=g).to(torch.bfloat16).to(dev) for h in (Hq, Hkv, Hkv))
        apply_rope(q, k, plan.positions, turns, magnitude=mag, q_out=q, k_out=k)
        impl.do_kv_cache_update(None, k, v, cache, plan.slot_mapping)
        kref.write(k.double().cpu().numpy(), plan.slot_mapping.tolist())
        vref.write(v.double().cpu().numpy(), plan.slot_mapping.tolist())
        md = PagedDecodeMetadata.from_plan(plan, tables, 192, num_decodes=decodes, max_query_len=max(new))
        rows = S if decodes is None else T + 2
        out = torch.zeros(rows, Hq * 128, dtype=torch.bfloat16, device=dev)
        impl.forward(None, q[:rows].reshape(rows, -1), None, None, cache, md, output=out)
        want = ref.sequences(q[:rows].double().cpu().numpy(), plan.query_start_loc.tolist(), lens.tolist(), kref.values(),
                             vref.values(), tables.tolist(), 1 / math.sqrt(128), True, 192)
        got = out.view(rows, Hq, 128).double().cpu().numpy()
        real = ~np.isnan(want).any(axis=(1, 2))
        assert real.sum() == T
        # (the bound of tests/test_gpu_paged8.py for bf16 and 192 tokens)
        lim = np.abs(vref.values()).max() * (2.0 ** -10 + 192 * 2.0 ** -25 + 2.0 ** -11.5) + 2.0 ** -8 * np.abs(want[real])
        assert np.all(np.abs(got[real] - want[real]) <= lim)
        # the same through the kernels' own entry points
        kc, vc = state.split_kv_cache(cache)
        if decodes is None:
            again = decode_paged8(q[:S], kc, state.k_format, vc, state.v_format, tables, lens, max_seq_len=192)
        else:
            again = prefill_paged8(q, plan.query_start_loc, kc, state.k_format, vc, state.v_format, tables, lens)
        assert np.all(np.abs(again.double().cpu().numpy()[real] - want[real]) <= lim)


def test_packed_layers_take_the_plan(dev):
    """The packed layers of the same step: plan_step's slots and tables through compress_paged_kv and decode."""
    Hq, Hkv, bs, S = 8, 2, 16, 2
    state = TurboQuantPagedState(128, device=dev, k_bits=4, block_size=bs)
    impl = TurboQuantPagedImpl(Hq, 128, 1 / math.sqrt(128), Hkv, state)
    cache = state.allocate_kv_cache(20, Hkv)
    ring, pool = new_pool(20, dev)
    tables = torch.full((S, 8), -1, dtype=torch.int32, device=dev)
    plan = plan_step(torch.zeros(S, dtype=torch.int32, device=dev), torch.tensor([33, 50], dtype=torch.int32, device=dev), tables,
                     ring, pool, bs, 83)
    k, v = (torch.randn(83, Hkv, 128, device=dev).to(torch.bfloat16) for _ in range(2))
    impl.do_kv_cache_update(None, k, v, cache, plan.slot_mapping)
    q = torch.randn(S, Hq, 128, device=dev).to(torch.bfloat16)
    out = torch.zeros(S, Hq * 128, dtype=torch.bfloat16, device=dev)
    impl.forward(None, q.view(S, -1), None, None, cache, PagedDecodeMetadata.from_plan(plan, tables, 128), output=out)
    for s, (a, b) in enumerate(((0, 33), (33, 83))):
        for h in range(Hq):
            sc = q[s, h].double() @ k[a:b, h // 4].double().T / math.sqrt(128)
            want = torch.softmax(sc, -1) @ v[a:b, h // 4].double()
            # 4-bit keys and values: a cosine distance of about 1 % on each side
            got = out.view(S, Hq, 128)[s, h].double()
            assert float((got - want).norm() / want.norm()) < 0.25
