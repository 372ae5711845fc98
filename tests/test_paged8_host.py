"""CPU tests of the 8-bit cache, rotary positions and step planning: formats, tiles, frequencies, refusals of the
Python entry points and of the C entries (which check on the host before any launch)."""

import math

import numpy as np
import pytest
import torch

import paged8_ref as ref
from turboquant import _lib
from turboquant.core.rope import rope_turns
from turboquant.integration.paged_backend import (PagedDecodeMetadata, TurboQuantPaged8State, TurboQuantPagedConfig,
                                                  TurboQuantPagedImpl, TurboQuantPagedState)
from turboquant.kernels import paged8, plan, rotation
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import Paged8Format, dequantize_paged8


def test_format():
    f = Paged8Format.for_keys("int8", 32)
    assert (f.code_bytes, f.tile_bytes) == (4096, 4112) and f.tile_bytes == _lib.lib().tq_kv8_tile_bytes(32)
    assert f == Paged8Format("int8", 32, "keys") and hash(f) == hash(Paged8Format("int8", 32))
    assert allocate_cache(3, 2, f).shape == (3, 2, 4112)
    for kw in (dict(encoding="e5m2"), dict(block_size=8), dict(block_size=0), dict(block_size=1 << 17), dict(layout="rows"),
               dict(head_dim=64)):
        with pytest.raises(ValueError):
            Paged8Format(**kw)
    assert _lib.lib().tq_kv8_tile_bytes(24) < 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("layout", ["keys", "values"])
def test_dequantize(code, layout):
    rng = np.random.default_rng(1)
    fmt = Paged8Format(code, 32, layout)
    val = ref.codes(rng.standard_normal((3, 2, 32, 128)) * 60, code)
    scale = 2.0 ** rng.integers(-9, 9, (3, 2))
    tile = ref.pack(val, scale, fmt)
    assert tile.shape[2] == fmt.tile_bytes
    np.testing.assert_array_equal(dequantize_paged8(tile, fmt).numpy(), val * scale[..., None, None])
    # the byte order that the C header states
    t, d = 21, 77
    at = (512 * (t // 4) + 4 * d + t % 4) if layout == "values" else 128 * t + d
    b = tile[1, 1, at:at + 1]
    got = b.view(torch.float8_e4m3fn if code == "e4m3" else torch.int8).float().item()
    assert got == val[1, 1, t, d]


def test_reference_codes():
    """The reference's e4m3 grid is torch's; its exponent is the smallest that holds the value."""
    y = np.concatenate([np.linspace(-448, 448, 4001), 2.0 ** np.arange(-12, 9) * 1.0625, [0.0, -0.0, 2.0 ** -10]])
    want = torch.from_numpy(y).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref.codes(y.astype(np.float32), "e4m3"), want)
    for code in ("e4m3", "int8"):
        for top in (1e-30, 0.3, 1.0, 7.0, 448.0, 448.1, 127.0, 127.5, 3e38):
            e = ref.exponent(top, code)
            assert top <= ref.TOP[code] * 2.0 ** e and (e == -126 or top > ref.TOP[code] * 2.0 ** (e - 1))


def test_rope_turns():
    t, m = rope_turns(64, theta=500.0)
    assert t.dtype == torch.float64 and m == 1.0
    np.testing.assert_allclose(t.numpy(), 500.0 ** (-np.arange(32) / 32) / (2 * np.pi), rtol=1e-14)
    lin, m = rope_turns(64, theta=500.0, scaling="linear", factor=4.0)
    np.testing.assert_allclose(lin.numpy(), t.numpy() / 4, rtol=1e-15)
    base, m = rope_turns(64, theta=500.0, scaling="base", factor=4.0)
    np.testing.assert_allclose([base[0].item(), base[-1].item()], [t[0].item(), t[-1].item() / 4], rtol=1e-12)
    parts, m = rope_turns(128, scaling="by_parts", factor=8.0, trained_length=4096)
    plain, _ = rope_turns(128)
    n = plain * 4096
    assert torch.equal(parts[n >= 32], plain[n >= 32]) and torch.allclose(parts[n <= 1], plain[n <= 1] / 8, rtol=1e-15)
    mid = (n > 1) & (n < 32)
    assert mid.any() and torch.all(parts[mid] < plain[mid]) and torch.all(parts[mid] > plain[mid] / 8)
    assert m == pytest.approx(0.1 * math.log(8) + 1)
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=130), dict(theta=0.0), dict(factor=-1.0), dict(scaling="x"),
               dict(scaling="base", rotary_dim=2), dict(scaling="by_parts", fast=1.0, slow=1.0),
               dict(scaling="by_parts", trained_length=0)):
        with pytest.raises(ValueError):
            rope_turns(**kw)


def test_cpu_tensors_are_refused():
    f, g = Paged8Format.for_keys(), Paged8Format.for_values()
    kc, vc = allocate_cache(2, 1, f), allocate_cache(2, 1, g)
    x, i = torch.zeros(1, 1, 128), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged8.quantize_paged8_kv(x, x, i, kc, vc, f, g)
    with pytest.raises(ValueError):
        paged8.decode_paged8(x, kc, f, vc, g, i[None], i)
    with pytest.raises(ValueError):
        paged8.prefill_paged8(x, torch.zeros(2, dtype=torch.int32), kc, f, vc, g, i[None], i)
    with pytest.raises(ValueError):
        rotation.apply_rope(x, None, i, rope_turns()[0])
    with pytest.raises(ValueError):
        plan.plan_step(i, i, i[None], i, torch.zeros(2, dtype=torch.int32), 16, 1)
    with pytest.raises(ValueError):
        plan.new_pool(0)
    ring, pool = plan.new_pool(3)
    assert ring.tolist() == [0, 1, 2] and pool.tolist() == [0, 3]


def test_protected_layers():
    cfg = TurboQuantPagedConfig(128, num_layers=6, num_protected_layers=1, k_bits=3, protected_bits=8, protected_encoding="int8",
                                block_size=32)
    st = cfg.get_state(0)
    assert isinstance(st, TurboQuantPaged8State) and st.k_format == Paged8Format.for_keys("int8", 32) and cfg.get_state(0) is st
    assert isinstance(cfg.get_state(2), TurboQuantPagedState)
    assert isinstance(TurboQuantPagedConfig(128, num_layers=6, protected_bits=4).get_state(0), TurboQuantPagedState)
    assert TurboQuantPagedConfig(128, num_layers=6).get_state(0) is None
    kv = st.allocate_kv_cache(5, 3)
    assert kv.shape == st.kv_cache_shape(5, 3) == TurboQuantPagedImpl.get_kv_cache_shape(5, 32, 3, 128, k_bits=8)
    k, v = st.split_kv_cache(kv)
    assert k.shape[2] == v.shape[2] == st.k_format.tile_bytes and v.data_ptr() - k.data_ptr() == st.k_format.tile_bytes
    with pytest.raises(ValueError):
        st.split_kv_cache(kv[..., :-1])
    with pytest.raises(ValueError):
        TurboQuantPaged8State(head_size=64)
    with pytest.raises(ValueError):
        TurboQuantPaged8State(encoding="int4")
    with pytest.raises(ValueError):
        TurboQuantPagedImpl.get_kv_cache_shape(5, 32, 3, 128, k_bits=8, v_bits=4)
    p = plan.StepPlan(torch.zeros(3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), None, None, None)
    md = PagedDecodeMetadata.from_plan(p, torch.zeros(2, 4, dtype=torch.int32), 64)
    assert md.query_start_loc is None and md.seq_lens is p.seq_lens
    assert PagedDecodeMetadata.from_plan(p, md.block_tables, 64, num_decodes=1).query_start_loc is p.query_start_loc


# ---- the C entries: every refusal comes from the host, before any launch ----

P = 4096  # a pointer that is never followed


def refused(name, fields, order, st, cases):
    fn = getattr(_lib.lib(), name)
    assert fn(None, None) == -1
    for change, code in cases:
        f = {**fields, **change}
        assert set(f) == set(order)
        assert fn(st.pack(*(f[k] for k in order)), None) == code, (change, code)


def test_c_update_refusals():
    order = ("k v kst ksh vst vsh kc vc ksb kch vsb vch slots tokens blocks dtype sdtype enc heads dim block").split()
    f = dict(k=P, v=P, kst=1024, ksh=128, vst=1024, vsh=128, kc=P, vc=P, ksb=4128, kch=2064, vsb=4128, vch=2064, slots=P, tokens=4,
             blocks=8, dtype=0, sdtype=4, enc=0, heads=2, dim=128, block=16)
    refused("tq_kv8_update", f, order, paged8._UPDATE, [
        (dict(dim=64), -2), (dict(block=0), -8), (dict(block=24), -8), (dict(dtype=3), -7), (dict(sdtype=0), -7), (dict(enc=2), -7),
        (dict(tokens=-1), -1), (dict(heads=-1), -1), (dict(blocks=-1), -1), (dict(k=0), -1), (dict(vc=0), -1), (dict(slots=0), -1),
        (dict(k=P + 2), -4), (dict(kst=1001), -4), (dict(kc=P + 8), -4), (dict(vsb=4120), -4), (dict(slots=P + 4), -4),
        (dict(tokens=1 << 40), -1), (dict(tokens=0, k=0), 0), (dict(heads=0, k=0), 0), (dict(blocks=0, k=0), 0)])


def test_c_attention_refusals():
    order = ("q out kc vc bt lens cu ws wsb qst qsh ost osh ksb ksh vsb vsh blocks bts qd od enc seqs hq hkv dim block mb msl mq "
             "flags sm zero").split()
    f = dict(q=P, out=P, kc=P, vc=P, bt=P, lens=P, cu=P, ws=P, wsb=1 << 40, qst=1024, qsh=128, ost=1024, osh=128, ksb=4128, ksh=2064,
             vsb=4128, vsh=2064, blocks=8, bts=4, qd=2, od=2, enc=1, seqs=2, hq=8, hkv=2, dim=128, block=16, mb=4, msl=64, mq=3, flags=1,
             sm=1.0, zero=0)
    common = [(dict(dim=64), -2), (dict(block=8), -8), (dict(qd=4), -7), (dict(od=-1), -7), (dict(enc=5), -7), (dict(seqs=-1), -1),
              (dict(hkv=0), -1), (dict(hq=0), -1), (dict(hq=7), -6), (dict(blocks=0), -1), (dict(blocks=1 << 40), -1), (dict(bts=3), -1),
              (dict(mb=-1), -1), (dict(sm=float("nan")), -1), (dict(sm=float("inf")), -1), (dict(q=P + 2), -4), (dict(ost=1001), -4),
              (dict(vc=P + 8), -4), (dict(ksb=4120), -4), (dict(q=0), -1), (dict(lens=0), -1), (dict(bt=0), -1), (dict(ws=0), -5),
              (dict(ws=P + 16), -5), (dict(wsb=16), -5), (dict(seqs=0, q=0), 0)]
    refused("tq_kv8_decode", f, order, paged8._ATTN, common + [(dict(hq=34), -6), (dict(msl=-1), -1)])
    refused("tq_kv8_prefill", f, order, paged8._ATTN, common + [(dict(cu=0), -1), (dict(mq=-1), -1), (dict(flags=2), -1),
                                                                (dict(mq=1 << 30), -1), (dict(mq=0, q=0), 0)])
    L = _lib.lib()
    assert L.tq_kv8_decode_workspace_bytes(4, 8, 3) == 0 and L.tq_kv8_decode_workspace_bytes(-1, 8, 2) == 0
    assert L.tq_kv8_prefill_workspace_bytes(2, 8, 8, 3, 4, 16) == 0 and L.tq_kv8_prefill_workspace_bytes(1, 1, 8, 2, 1, 16) > 0


def test_c_rope_refusals():
    order = ("q k qo ko qst qsh kst ksh qost qosh kost kosh pos turns tokens dtype pd hq hk dim rot inter mag").split()
    f = dict(q=P, k=P, qo=2 * P, ko=2 * P, qst=1024, qsh=128, kst=256, ksh=128, qost=1024, qosh=128, kost=256, kosh=128, pos=P, turns=P,
             tokens=3, dtype=2, pd=3, hq=8, hk=2, dim=128, rot=128, inter=0, mag=1.0)
    refused("tq_rope", f, order, rotation._ROPE, [
        (dict(dim=64), -2), (dict(dtype=4), -7), (dict(pd=2), -7), (dict(tokens=-1), -1), (dict(rot=0), -1), (dict(rot=3), -1),
        (dict(rot=130), -1), (dict(hq=-1), -1), (dict(q=0), -1), (dict(ko=0), -1), (dict(pos=0), -1), (dict(turns=0), -1),
        (dict(q=P + 1), -4), (dict(turns=P + 4), -4), (dict(pos=P + 2), -4), (dict(pd=4, pos=P + 4), -4),
        (dict(qo=P, qost=2048), -1), (dict(tokens=0, q=0), 0), (dict(hq=0, hk=0, q=0), 0)])


def test_c_plan_refusals():
    order = ("past new tables ts ring pin pout lens start pos slots ws wsb tokens seqs width blocks bs").split()
    f = dict(past=P, new=P, tables=P, ts=8, ring=P, pin=P, pout=P, lens=P, start=P, pos=P, slots=P, ws=P, wsb=1 << 30, tokens=9, seqs=3,
             width=8, blocks=64, bs=16)
    refused("tq_plan_step", f, order, plan._PLAN, [
        (dict(bs=0), -8), (dict(bs=20), -8), (dict(seqs=-1), -1), (dict(seqs=(1 << 20) + 1), -1), (dict(tokens=-1), -1),
        (dict(tokens=1 << 31), -1), (dict(blocks=0), -1), (dict(width=1 << 28, ts=1 << 28), -1), (dict(ts=7), -1), (dict(past=0), -1),
        (dict(ring=0), -1), (dict(pout=0), -1), (dict(start=0), -1), (dict(slots=0), -1), (dict(ws=0), -5), (dict(ws=P + 8), -5),
        (dict(wsb=8), -5)])
    assert _lib.lib().tq_plan_step_workspace_bytes(-1) == 0


def test_c_launch_limits():
    """Calls whose launches would have 2^32 threads or more."""
    order = ("q out kc vc bt lens cu ws wsb qst qsh ost osh ksb ksh vsb vsh blocks bts qd od enc seqs hq hkv dim block mb msl mq "
             "flags sm zero").split()
    f = dict(q=P, out=P, kc=P, vc=P, bt=P, lens=P, cu=P, ws=P, wsb=1 << 40, qst=1024, qsh=128, ost=1024, osh=128, ksb=4128, ksh=2064,
             vsb=4128, vsh=2064, blocks=8, bts=4, qd=2, od=2, enc=1, seqs=1 << 18, hq=64, hkv=4, dim=128, block=16, mb=4, msl=64, mq=3,
             flags=1, sm=1.0, zero=0)
    refused("tq_kv8_decode", f, order, paged8._ATTN, [(dict(), -1)])
    order = ("q k qo ko qst qsh kst ksh qost qosh kost kosh pos turns tokens dtype pd hq hk dim rot inter mag").split()
    f = dict(q=P, k=P, qo=2 * P, ko=2 * P, qst=1024, qsh=128, kst=256, ksh=128, qost=1024, qosh=128, kost=256, kosh=128, pos=P, turns=P,
             tokens=1 << 27, dtype=2, pd=3, hq=8, hk=2, dim=128, rot=128, inter=0, mag=1.0)
    refused("tq_rope", f, order, rotation._ROPE, [(dict(), -1)])
