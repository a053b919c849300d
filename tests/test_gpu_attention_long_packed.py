"""Packed tensors of more than 2^31 elements: the sequence at their end gets what it gets alone."""
import pytest
import torch

import periodicdent42_b200 as bsk

pytestmark = pytest.mark.gpu


def test_last_sequence(no_device_error, cuda_dev):
    H, G, D, n = 64, 8, 128, 55
    lens = [2048] * 128 + [n]
    T = sum(lens)
    assert (T - n) * H * D >= 2 ** 31 and T * H * D > 2 ** 31
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q = torch.zeros(T, H, D, dtype=torch.bfloat16, device=cuda_dev)
    k, v = (torch.zeros(T, G, D, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    for t in (q, k, v):
        t[-n:] = torch.randn(n, *t.shape[1:], generator=g, device=cuda_dev)
    do = torch.zeros_like(q)
    do[-n:] = torch.randn(n, H, D, generator=g, device=cuda_dev)
    cu = torch.tensor([0] + lens, device=cuda_dev).cumsum(0)

    def run(q, k, v, do, cu):
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = bsk.attention_varlen(*x, cu)
        return (o.detach(), *torch.autograd.grad(o, x, do))

    got = run(q, k, v, do, cu)
    want = run(*(t[-n:].contiguous() for t in (q, k, v, do)), torch.tensor([0, n], device=cuda_dev))
    assert all(torch.equal(a[-n:], b) for a, b in zip(got, want))
    pos = torch.arange(T, device=cuda_dev)
    f = bsk.rotary_frequencies(D, device=cuda_dev)[0]
    for inter in (False, True):
        a, b = bsk.rotary_embedding(q, k, pos, f, interleaved=inter)
        wa, wb = bsk.rotary_embedding(q[-n:].contiguous(), k[-n:].contiguous(), pos[-n:], f, interleaved=inter)
        assert torch.equal(a[-n:], wa) and torch.equal(b[-n:], wb)
        del a, b
