"""Rotary angles at far positions against exact arithmetic: whole turns are dropped without an error at any 64-bit position."""
import math
from fractions import Fraction

import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu
INV_2PI = Fraction("0.15915494309189533576888376337251436203445964574045644874766734405889679763422653509")
FAR = [0, 1, 2 ** 27 + 5, 2 ** 31 - 1, -(2 ** 31), 2 ** 33 + 3, 2 ** 40 + 3, -(2 ** 45) - 11, 2 ** 53 + 1, 2 ** 60 + 12345, 2 ** 63 - 1, 2 ** 63 - 100,
       -(2 ** 63), 100 - 2 ** 63]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("backward", [False, True])
def test_far_positions(no_device_error, cuda_dev, dtype, backward):
    D = 64
    f = bsk.rotary_frequencies(D, device=cuda_dev)[0]
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    x = torch.randn(len(FAR), 2, D, generator=g, device=cuda_dev).to(dtype)
    pos = torch.tensor(FAR, device=cuda_dev)
    if backward:
        leaf = torch.zeros_like(x).requires_grad_(True)
        (got,) = torch.autograd.grad(bsk.rotary_embedding(leaf, None, pos, f)[0], leaf, x)
    else:
        got = bsk.rotary_embedding(x, None, pos, f)[0]
    turn = torch.empty(len(FAR), D // 2, dtype=torch.float64)
    for i, p in enumerate(FAR):
        for j, fj in enumerate(f.tolist()):
            t = p * Fraction(fj) * INV_2PI
            turn[i, j] = float(t - round(t))
    angle = (turn * (2 * math.pi) * (-1 if backward else 1))[:, None].to(cuda_dev)
    a, b = x.double()[..., :D // 2], x.double()[..., D // 2:]
    want = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)
    # as in the other rotary tests: the result's rounding, and 2^-20 of |a| + |b| for cosine, sine and the products
    size = x.double().abs().amax(-1, keepdim=True) * 2
    assert pa.worst(got, want, pa.half_step(dtype) * want.abs() + 2.0 ** -20 * size) <= 1.0
