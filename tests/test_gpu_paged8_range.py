"""8-bit paged attention at the ends of its number ranges: values far from 1."""

import pytest
import torch

from test_gpu_paged8 import bound
from test_gpu_paged8_edges import causal64, filled
from turboquant.kernels.paged8 import decode_paged8, prefill_paged8

pytestmark = pytest.mark.gpu


def attend(entry, q, args, seqs, n, **kw):
    """Rows q [T, Hq, 128], the last tokens of seqs sequences of n tokens that share one table."""
    kc, kf, vc, vf, bt = args
    sl = torch.full((seqs,), n, dtype=torch.int32, device=q.device)
    bt = bt.expand(seqs, -1).contiguous()
    if entry == "decode":
        return decode_paged8(q, kc, kf, vc, vf, bt, sl, **kw)
    cu = torch.arange(0, q.shape[0] + 1, q.shape[0] // seqs, dtype=torch.int32, device=q.device)
    return prefill_paged8(q, cu, kc, kf, vc, vf, bt, sl, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("entry", ["decode", "prefill"])
@pytest.mark.parametrize("past,power", [(10, 100), (6000, 70), (6000, 100), (6000, 121), (6000, -60)])
def test_values_of_any_size(dev, entry, code, dtype, past, power):
    """Values near the ends of fp32's range, of a sequence that one wave takes and of a cut one."""
    g = torch.Generator(device=dev).manual_seed(past + power)
    new = 1 if entry == "decode" else 20
    k, v = (torch.randn(past + new, 2, 128, generator=g, device=dev) for _ in range(2))
    args, kval, vval = filled(k, v * 2.0 ** power, code, 16, dev)
    q = torch.randn(new, 8, 128, generator=g, device=dev).to(dtype)
    got = attend(entry, q, args, 1, past + new).double().cpu().numpy()
    want = causal64(q, kval, vval, past).cpu().numpy()
    lim = bound(float(vval.abs().max()), past + new, dtype, dtype, want)
    assert (abs(got - want) <= lim).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("entry", ["decode", "prefill"])
@pytest.mark.parametrize("seqs,power", [(300, 113), (512, 113), (300, 85)])
def test_sums_of_large_values(dev, entry, code, dtype, seqs, power):
    """The mean of 30000 values of one sign, whose plain sum passes fp32's range: 300 sequences of 4 heads are cut, 512 are
    not.  (1000 steps added one after the other: 2^-14 of the sum, within the bound's share for scores, all 0 here.)"""
    n = 30000
    g = torch.Generator(device=dev).manual_seed(seqs)
    v = 1 + torch.rand(n, 4, 128, generator=g, device=dev)
    args, _, vval = filled(torch.zeros_like(v), v * 2.0 ** power, code, 16, dev)
    q = torch.randn(seqs, 4, 128, generator=g, device=dev).to(dtype)
    got = attend(entry, q, args, seqs, n).double().cpu().numpy()
    want = vval.mean(0).cpu().numpy()[None]
    assert (abs(got - want) <= bound(float(vval.abs().max()), n, dtype, dtype, want)).all()
