"""Destinations whose rows share memory are refused; sources may."""

import pytest
import torch

from test_gpu_paged8 import formats
from turboquant.core.rope import rope_turns
from turboquant.kernels.paged import allocate_cache
from turboquant.kernels.paged8 import decode_paged8, prefill_paged8
from turboquant.kernels.rotation import apply_rope

pytestmark = pytest.mark.gpu


def test_rope(dev):
    turns, _ = rope_turns(128, device=dev)
    pos = torch.arange(5, dtype=torch.int32, device=dev)
    one = torch.randn(5, 1, 128, device=dev)
    heads, tokens = one.expand(5, 3, 128), one[:1].expand(5, 1, 128)
    for x in (heads, tokens):
        with pytest.raises(ValueError):
            apply_rope(x, None, pos, turns, q_out=x)
        with pytest.raises(ValueError):
            apply_rope(one, x, pos, turns, k_out=x)
        assert torch.equal(apply_rope(x, None, pos, turns)[0], apply_rope(x.contiguous(), None, pos, turns)[0])
    alone = one.as_strided((5, 1, 128), (128, 0, 1))      # (one head: its stride says nothing)
    want = apply_rope(one, None, pos, turns)[0]
    assert torch.equal(apply_rope(alone, None, pos, turns, q_out=alone)[0], want)


def test_attention(dev):
    kf, vf = formats("e4m3", 16)
    args = (allocate_cache(4, 1, kf, device=dev), kf, allocate_cache(4, 1, vf, device=dev), vf,
            torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev))
    q = torch.randn(2, 4, 128, device=dev)
    cu = torch.arange(3, dtype=torch.int32, device=dev)
    for out in (q[:, :1].expand(2, 4, 128), q[:1].expand(2, 4, 128)):
        with pytest.raises(ValueError):
            decode_paged8(q, *args, out=out)
        with pytest.raises(ValueError):
            prefill_paged8(q, cu, *args, out=out)
    assert torch.equal(decode_paged8(q[:, :1].expand(2, 4, 128), *args), decode_paged8(q[:, :1].repeat(1, 4, 1), *args))
