"""8-bit paged attention at the ends of its number ranges: many small probabilities, values far from 1."""

import math

import pytest
import torch

from test_gpu_paged8 import HALF, bound
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("entry,down", [("decode", 26.5), ("decode", 20.5), ("prefill", 17.5)])
@pytest.mark.parametrize("seqs,at", [(1, 15000), (512, 0), (512, 15000)])
def test_small_probabilities_add_up(dev, entry, down, code, dtype, seqs, at):
    """One token's probability is 2^down times that of each of 29999 others, which alone have values in dims 64 and up:
    outputs there are the sum of the small ones.  (512 sequences of 4 heads: a wave has all tokens of one.)

    All small probabilities are one number; as normal fp16 numbers they are off by 2^-11 of it, the large one by as
    much.  Scores are single products, exact but for three factors' roundings: 27 * 2^-22 in log2 units, below 2^-17.  A
    wave adds its at most 940 steps one after the other, 940 * 2^-24 of rounding at most in either sum, or 470 waves'
    pieces are joined: below 2^-13 together.  Then the output's own rounding."""
    n = 30000
    k, v = (torch.zeros(n, 4, 128, device=dev) for _ in range(2))
    k[at, :, 9] = 1.0
    v[:, :, 64:] = 1.0
    v[at] = 0.0
    v[at, :, :64] = 1.0
    args, _, _ = filled(k, v, code, 16, dev)
    q = torch.zeros(seqs, 4, 128, dtype=dtype, device=dev)
    q[..., 9] = 1.0
    got = attend(entry, q, args, seqs, n, sm_scale=down * math.log(2)).double()
    tail = (n - 1) * 2.0 ** -down
    want = torch.full((128,), 1 / (1 + tail), dtype=torch.float64, device=dev)
    want[64:] = tail / (1 + tail)
    lim = want * (2 * 2.0 ** -11 + 2.0 ** -13 + 2.0 ** -17 + HALF[dtype])
    assert torch.all((got - want).abs() <= lim), float(((got - want).abs() / want).max())


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("entry", ["decode", "prefill"])
def test_small_probabilities_in_fp32(dev, entry, code):
    """As above in fp32, where a probability is the sum of two fp16 numbers: off by half of their smallest step, 2^-25,
    with the largest at 2^10 or more.  The small ones are 2^-18 of that, half a step between two numbers of a scale with the
    largest at 2^4: 2^-18 of them.  Scores: 19 * 2^-22, below 2^-17.  125 steps' sums, twice: 2^-16.  The fp32 output."""
    n, seqs, down = 4000, 512, 28 - math.log2(1000.5)
    k, v = (torch.zeros(n, 4, 128, device=dev) for _ in range(2))
    k[0, :, 9] = 1.0
    v[:, :, 64:] = 1.0
    v[0] = 0.0
    args, _, _ = filled(k, v, code, 16, dev)
    q = torch.zeros(seqs, 4, 128, device=dev)
    q[..., 9] = 1.0
    got = attend(entry, q, args, seqs, n, sm_scale=down * math.log(2)).double()[..., 64:]
    tail = (n - 1) * 2.0 ** -down
    want = tail / (1 + tail)
    assert float((got / want - 1).abs().max()) <= 2.0 ** -18 + 2.0 ** -17 + 2.0 ** -16 + 2.0 ** -24


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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("entry", ["decode", "prefill"])
@pytest.mark.parametrize("power", [20, 21, 22, 23, 24, 25, 26, 27, 28, 30, 40, 70, 110, 120])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(dev, entry, code, dtype, power, sign):
    """Scores of about 2^power in log2 units, of either sign, whose largest several tokens share: the mean of these tokens' values.
    (The others lie 2^-6 of that lower, 2^14 in log2 units and more, so that nothing of them is left.)  A short sequence, and
    a cut one with the largest in its middle and at its end."""
    g = torch.Generator(device=dev).manual_seed(power)
    for n, at in ((70, (3, 40, 69)), (5000, (2100, 2111, 4999)), (70, (0, 1))):
        k = torch.zeros(n, 2, 128, device=dev)
        k[:, :, 9] = 1.0 if sign > 0 else 1.0 + 2.0 ** -2      # (exact in e4m3 and, with the block's scale, in int8)
        for t in at:
            k[t, :, 9] = 1.0 + 2.0 ** -2 if sign > 0 else 1.0
        k *= sign * 2.0 ** (power // 2)
        v = torch.randn(n, 2, 128, generator=g, device=dev)
        args, kval, vval = filled(k, v, code, 16, dev)
        assert torch.equal(kval, k.double())
        q = torch.zeros(1, 8, 128, dtype=dtype, device=dev)
        # seven bits of mantissa, other ones in each head
        q[..., 9] = (1.0 + torch.arange(8, device=dev) * 15 / 128) * 2.0 ** (power - power // 2)
        got = attend(entry, q, args, 1, n, sm_scale=1.0 / 1.7).double()
        want = vval[list(at)].mean(0).repeat_interleave(4, 0)[None].cpu().numpy()
        lim = bound(float(vval.abs().max()), n, dtype, dtype, want)
        assert (abs(got.cpu().numpy() - want) <= lim).all(), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("past", [0, 6000])
def test_far_and_near_scores_side_by_side(dev, code, dtype, past):
    """Rows of ordinary scores among rows of far ones, which from token 32 on pass from the first kind to the second.  (Far scores leave the largest one alone: the bound's share for scores is
    2^-24 of a score, and two of them lie that close in no row, as is checked.)"""
    g = torch.Generator(device=dev).manual_seed(past + 3)
    new = 75
    k, v = (torch.randn(past + new, 2, 128, generator=g, device=dev) for _ in range(2))
    k[:32] *= 2.0 ** -32
    args, kval, vval = filled(k, v, code, 16, dev)
    q = torch.randn(new, 8, 128, generator=g, device=dev)
    far = torch.arange(new, device=dev) % 3 == 1
    far[[40, 41, 42, 74]] = True
    q[far] *= 2.0 ** 34
    q = q.to(dtype)
    for entry in ("prefill", "decode"):
        if entry == "prefill":
            got, want, n = attend(entry, q, args, 1, past + new), causal64(q, kval, vval, past), past + new
            s = torch.matmul(q.double().transpose(0, 1), kval.repeat_interleave(4, 1).permute(1, 2, 0)) / math.sqrt(128)
            s.masked_fill_(torch.arange(n, device=dev) > past + torch.arange(new, device=dev)[:, None], -math.inf)
            top = s[:, far].topk(2, -1).values if past else s[:, far & (torch.arange(new, device=dev) > 33)].topk(2, -1).values
            assert float((top[..., 0] - top[..., 1]).min()) > 2.0 ** 12
        else:
            row = q[-1:]
            got, want = attend(entry, row, args, 1, past + new), causal64(row, kval, vval, past + new - 1)
        w = want.cpu().numpy()
        assert (abs(got.double().cpu().numpy() - w) <= bound(float(vval.abs().max()), past + new, dtype, dtype, w)).all()
