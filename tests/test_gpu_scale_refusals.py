"""Softmax and rotary scales that the kernels cannot use are refused as argument errors, those next to them taken."""
import math

import pytest
import torch

import periodicdent42_b200 as bsk

pytestmark = pytest.mark.gpu


def test_attention_scales(no_device_error, cuda_dev):
    q, k, v = (torch.randn(8, h, 64, device=cuda_dev).bfloat16() for h in (4, 2, 2))
    c = [torch.randn(1, 16, 2, 64, device=cuda_dev).bfloat16() for _ in range(2)]
    at = (torch.tensor([[0]], device=cuda_dev), torch.tensor([8], device=cuda_dev), torch.tensor([0, 8], device=cuda_dev))
    for call in (lambda s: bsk.attention_varlen(q, k, v, at[2], scale=s), lambda s: bsk.attention_paged(q, *c, *at, scale=s),
                 lambda s: bsk.attention_varlen(q.clone().requires_grad_(True), k, v, at[2], scale=s)):
        for bad in (0.0, -1.0, 1e-60, 1e30, 1e40, math.inf, math.nan):
            with pytest.raises(ValueError, match="scale"):
                call(bad)
        assert torch.isfinite(call(1e-30)).all()


def test_rotary_scales(no_device_error, cuda_dev):
    q = torch.randn(4, 2, 64, device=cuda_dev)
    pos, f = torch.arange(4, device=cuda_dev), bsk.rotary_frequencies(64, device=cuda_dev)[0]
    for bad in (math.inf, -math.inf, math.nan, 1e30):
        with pytest.raises(ValueError, match="scale"):
            bsk.rotary_embedding(q, None, pos, f, scale=bad)
    assert torch.equal(bsk.rotary_embedding(q, None, pos, f, scale=-1.0)[0], -bsk.rotary_embedding(q, None, pos, f)[0])
