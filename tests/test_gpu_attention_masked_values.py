"""Finite values as large as bfloat16 holds, of keys that a row does not see or that lie far below its best: weight zero."""
import pytest
import torch

import periodicdent42_b200 as bsk

pytestmark = pytest.mark.gpu
LARGE = 2.0 ** 127


@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (3, 1, 128)])
def test_packed(no_device_error, cuda_dev, H, G, D):
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q, k, v = (torch.randn(300, h, D, generator=g, device=cuda_dev).bfloat16() for h in (H, G, G))
    cu = torch.tensor([0, 300], device=cuda_dev)
    want = bsk.attention_varlen(q, k, v, cu)
    for first in (33, 150, 299):
        big = v.clone()
        big[first:] = LARGE
        assert torch.equal(bsk.attention_varlen(q, k, big, cu)[:first], want[:first])
    k[200:] = -k[200:].abs()  # keys 200.. : scores some hundreds below the others
    q.copy_(q.abs() * 32 + 32)
    k[:200] = 0
    want = bsk.attention_varlen(q, k, v, cu, causal=False)
    v[200:] = LARGE
    assert torch.equal(bsk.attention_varlen(q, k, v, cu, causal=False), want)


@pytest.mark.parametrize("new", [3, 150])  # either kernel
def test_paged(no_device_error, cuda_dev, new):
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q = torch.randn(new, 4, 64, generator=g, device=cuda_dev).bfloat16()
    k, v = (torch.randn(25, 16, 2, 64, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    at = (torch.arange(25, device=cuda_dev)[None], torch.tensor([400], device=cuda_dev), torch.tensor([0, new], device=cuda_dev))
    want = bsk.attention_paged(q, k, v, *at)
    v.view(400, 2, 64)[399] = LARGE
    assert torch.equal(bsk.attention_paged(q, k, v, *at)[:-1], want[:-1])


@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (3, 1, 128)])
def test_gradients(no_device_error, cuda_dev, H, G, D):
    """A value or an output's gradient so large that their product overflows does not reach rows that do not see it: dQ of the
    rows before the value, dK of the keys behind the row."""
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q, do = (torch.randn(300, H, D, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    k, v = (torch.randn(300, G, D, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    cu = torch.tensor([0, 300], device=cuda_dev)

    def grads(v, do):
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(bsk.attention_varlen(*x, cu), x, do)

    want = grads(v, do)
    for at in (33, 150, 299):
        big = v.clone()
        big[at] = LARGE
        assert torch.equal(grads(big, do)[0][:at], want[0][:at])
        big = do.clone()
        big[at] = LARGE
        got = grads(v, big)
        assert torch.equal(got[1][at + 1:], want[1][at + 1:]) and torch.equal(got[2][at + 1:], want[2][at + 1:])
