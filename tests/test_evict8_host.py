"""CPU tests of windows with sinks, accumulated weights and eviction: refusals of the Python entry points and of the C entries (which
check on the host before any launch), layer configuration, and the plain implementations against brute force."""

import struct

import numpy as np
import pytest
import torch

import evict8_ref as eref
from turboquant import _lib
from turboquant.integration.paged_backend import TurboQuantPaged8State, TurboQuantPagedImpl, TurboQuantPagedState
from turboquant.kernels import evict8, paged8
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import Paged8Format

P = 4096  # a pointer that is never followed
ATTN = ("q out kc vc bt lens cu ws wsb qst qsh ost osh ksb ksh vsb vsh blocks bts qd od enc seqs hq hkv dim block mb msl mq "
        "flags sm zero").split()
REACH = "mass msb msh window sinks last rest".split()
WINDOW = struct.Struct(paged8._ATTN.format + paged8._REACH.format[1:])
EVICT = ("kc vc mass bt lens change ws wsb ksb ksh vsb vsh msb msh blocks bts enc seqs hkv dim block mb msl keep recent sinks "
         "longer rest").split()


def refused(name, fields, order, st, cases):
    fn = getattr(_lib.lib(), name)
    assert fn(None, None) == -1
    for change, code in cases:
        f = {**fields, **change}
        assert set(f) == set(order)
        assert fn(st.pack(*(f[k] for k in order)), None) == code, (change, code)


def attn(**kw):
    f = dict(q=P, out=P, kc=P, vc=P, bt=P, lens=P, cu=P, ws=P, wsb=1 << 40, qst=1024, qsh=128, ost=1024, osh=128, ksb=4128, ksh=2064,
             vsb=4128, vsh=2064, blocks=8, bts=4, qd=2, od=2, enc=1, seqs=2, hq=8, hkv=2, dim=128, block=16, mb=4, msl=64, mq=3, flags=1,
             sm=1.0, zero=0, mass=P, msb=32, msh=16, window=20, sinks=4, last=2, rest=0)
    return {**f, **kw}


COMMON = [(dict(dim=64), -2), (dict(block=8), -8), (dict(qd=4), -7), (dict(enc=5), -7), (dict(seqs=-1), -1), (dict(hkv=0), -1),
          (dict(hq=7), -6), (dict(blocks=0), -1), (dict(bts=3), -1), (dict(mb=-1), -1), (dict(sm=float("nan")), -1),
          (dict(q=P + 2), -4), (dict(kc=P + 8), -4), (dict(ksb=4120), -4), (dict(q=0), -1), (dict(lens=0), -1), (dict(bt=0), -1),
          (dict(ws=0), -5), (dict(ws=P + 16), -5), (dict(wsb=16), -5), (dict(seqs=0, q=0), 0), (dict(window=-1), -1),
          (dict(sinks=-1), -1), (dict(window=0), -1), (dict(rest=1), -1)]
MASS = [(dict(mass=P + 4), -4), (dict(msb=30), -4), (dict(msh=17), -4)]


def test_c_window_refusals():
    refused("tq_kv8_decode_window", attn(), ATTN + REACH, WINDOW, COMMON + MASS + [
        (dict(hq=34), -6), (dict(msl=-1), -1), (dict(out=0), -1), (dict(vc=0), -1)])
    refused("tq_kv8_prefill_window", attn(mass=0), ATTN + REACH, WINDOW, COMMON + [
        (dict(cu=0), -1), (dict(mq=-1), -1), (dict(flags=2), -1), (dict(flags=0), -1), (dict(mass=P), -1), (dict(mq=0, q=0), 0)])
    refused("tq_kv8_observe", attn(out=0, vc=0), ATTN + REACH, WINDOW, COMMON + MASS + [
        (dict(mass=0), -1), (dict(cu=0), -1), (dict(mq=-1), -1), (dict(msl=-1), -1), (dict(flags=0), -1), (dict(flags=3), -1),
        (dict(last=0), -1), (dict(mq=0, q=0), 0), (dict(msl=0, q=0), 0)])


def test_c_window_workspaces():
    L = _lib.lib()
    plain = L.tq_kv8_decode_workspace_bytes(4, 8, 2)
    assert L.tq_kv8_decode_window_workspace_bytes(4, 8, 2, 1000, 0, 0, 0) == plain
    full = L.tq_kv8_decode_window_workspace_bytes(4, 8, 2, 1000, 0, 0, 1)
    assert full >= plain + 4 * 8 * 1000 * 4
    # a window's scores alone, and not more than all
    assert plain < L.tq_kv8_decode_window_workspace_bytes(4, 8, 2, 1000, 64, 4, 1) < full
    assert L.tq_kv8_decode_window_workspace_bytes(4, 8, 2, 1000, 2000, 4, 1) == full
    # exactly what the entry asks for (the next check behind it is a device, which is not here: so only too little is shown)
    f = attn(wsb=L.tq_kv8_decode_window_workspace_bytes(2, 8, 2, 64, 20, 4, 1) - 1)
    assert L.tq_kv8_decode_window(WINDOW.pack(*(f[k] for k in ATTN + REACH)), None) == -5
    assert L.tq_kv8_observe_workspace_bytes(2, 8, 0, 8, 2, 2, 64) == 0 == L.tq_kv8_observe_workspace_bytes(2, 8, 3, 8, 3, 2, 64)
    assert L.tq_kv8_observe_workspace_bytes(1, 8, 3, 8, 2, 2, 64) > 0 == L.tq_kv8_observe_workspace_bytes(1, 8, 3, 8, 2, 2, 0)
    assert L.tq_kv8_evict_workspace_bytes(2, 2, 0, 16) == 0 == L.tq_kv8_evict_workspace_bytes(2, 2, 8, 24)
    assert L.tq_kv8_evict_workspace_bytes(1, 1, 1, 16) > 0


def test_c_evict_refusals():
    f = dict(kc=P, vc=P, mass=P, bt=P, lens=P, change=P, ws=P, wsb=1 << 40, ksb=4128, ksh=2064, vsb=4128, vsh=2064, msb=32, msh=16,
             blocks=8, bts=4, enc=1, seqs=2, hkv=2, dim=128, block=16, mb=4, msl=64, keep=40, recent=8, sinks=2, longer=48, rest=0)
    refused("tq_kv8_evict", f, EVICT, evict8._EVICT, [
        (dict(dim=64), -2), (dict(block=0), -8), (dict(block=24), -8), (dict(enc=2), -7), (dict(seqs=-1), -1), (dict(hkv=0), -1),
        (dict(blocks=0), -1), (dict(blocks=1 << 40), -1), (dict(bts=3), -1), (dict(mb=-1), -1), (dict(msl=-1), -1), (dict(keep=0), -1),
        (dict(recent=-1), -1), (dict(sinks=-1), -1), (dict(recent=39), -1), (dict(longer=39), -1), (dict(rest=1), -1),
        (dict(kc=P + 8), -4), (dict(mass=P + 4), -4), (dict(vsb=4120), -4), (dict(msh=18), -4), (dict(kc=0), -1), (dict(mass=0), -1),
        (dict(bt=0), -1), (dict(lens=0), -1), (dict(change=0), -1), (dict(ws=0), -5), (dict(ws=P + 8), -5), (dict(wsb=64), -5),
        (dict(seqs=1 << 22, hkv=2), -1), (dict(seqs=0, kc=0), 0)])


def test_cpu_tensors_are_refused():
    f, g = Paged8Format.for_keys(), Paged8Format.for_values()
    kc, vc, mass = allocate_cache(2, 1, f), allocate_cache(2, 1, g), evict8.allocate_mass(2, 1, 16)
    x, i = torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.int32)
    assert mass.shape == (2, 1, 16) and mass.dtype == torch.float32 and not mass.any()
    with pytest.raises(ValueError):
        paged8.decode_paged8(x, kc, f, vc, g, i[None], i, window=4, mass=mass)
    with pytest.raises(ValueError):
        evict8.observe_paged8(x, torch.zeros(2, dtype=torch.int32), kc, f, i[None], i, mass)
    with pytest.raises(ValueError):
        evict8.evict_paged8(kc, f, vc, g, mass, i[None], i, 4)


def test_impl():
    st = TurboQuantPaged8State(128, block_size=32)
    assert st.allocate_mass(3, 2).shape == (3, 2, 32)
    impl = TurboQuantPagedImpl(8, 128, 0.1, 2, st, sliding_window=100, sinks=4, mass=st.allocate_mass(3, 2))
    assert impl.reach == dict(window=100, sinks=4) and TurboQuantPagedImpl(8, 128, 0.1, 2, st).reach == {}
    packed = TurboQuantPagedState(128)
    assert TurboQuantPagedImpl(8, 128, 0.1, 2, packed).mass is None
    for kw in (dict(sliding_window=100), dict(mass=st.allocate_mass(3, 2))):
        with pytest.raises(ValueError):
            TurboQuantPagedImpl(8, 128, 0.1, 2, packed, **kw)
    for kw in (dict(sinks=4), dict(sliding_window=0), dict(sliding_window=4, sinks=-1), dict(observe_last=0)):
        with pytest.raises(ValueError):
            TurboQuantPagedImpl(8, 128, 0.1, 2, st, **kw)


def test_mass_checks():
    for t in (torch.zeros(2, 3, 16, dtype=torch.float64), torch.zeros(2, 3, 32), torch.zeros(2, 16), torch.zeros(2, 3, 32)[..., ::2],
              torch.zeros(2, 1, 16).expand(2, 3, 16), torch.zeros(1, 3, 16).expand(2, 3, 16), torch.zeros(200)[1:97].view(2, 3, 16),
              torch.zeros(200).as_strided((2, 3, 16), (17, 34, 1)), torch.zeros(200).as_strided((2, 3, 16), (16, 16, 1))):
        with pytest.raises(ValueError):
            paged8._check_mass(t, 2, 3, 16)
    assert paged8._check_mass(torch.zeros(2, 3, 16), 2, 3, 16) == (48, 16)
    assert paged8._check_mass(torch.zeros(3, 2, 16).transpose(0, 1), 2, 3, 16) == (16, 32)
    assert paged8._check_mass(torch.zeros(2, 5, 20)[:, 1:4, :16], 2, 3, 16) == (100, 20)
    for w, s in ((None, 1), (0, 0), (-3, 0), (4, -1)):
        with pytest.raises(ValueError):
            paged8._check_window(w, s)
    assert paged8._check_window(None, 0) == (0, 0) and paged8._check_window(1 << 40, 2) == (0x7fffffff, 2)


def test_reference():
    """The plain choice of tokens against an ordering by hand, and the window against its definition."""
    nan = float("nan")
    m = np.array([9.0, 1.0, 5.0, nan, -0.0, 0.0, 5.0, 5.0, 2.0, 3.0])
    ok = np.ones(10, dtype=bool)
    assert eref.chosen(m, ok, 10, 6, 2, 1) == [0, 2, 6, 7, 8, 9]
    assert eref.chosen(m, ok, 10, 8, 2, 1) == [0, 1, 2, 4, 6, 7, 8, 9]          # -0 and 0 tie: the earlier one
    assert eref.chosen(m, ok, 10, 9, 1, 0) == [0, 1, 2, 4, 5, 6, 7, 8, 9]
    ok[2] = False
    assert eref.chosen(m, ok, 10, 7, 2, 1) == [0, 1, 4, 6, 7, 8, 9]
    for L in (1, 5, 40):
        for w in (None, 1, 3, 50):
            for sinks in (0, 2):
                for p in range(L):
                    see = [t <= p and (w is None or t > p - w or t < sinks) for t in range(L)]
                    assert eref.visible(p, L, w, sinks).tolist() == see
