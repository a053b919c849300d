"""Rotary positions against their 64-bit definition: layouts, partial heads, types, strides, far and negative positions,
gradients, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu


def _make(T, H, G, D, r, dtype, dev, far=100000, seed=0, pos_dtype=torch.int64):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(T, H, D, generator=g, device=dev).to(dtype)
    k = torch.randn(T, G, D, generator=g, device=dev).to(dtype)
    pos = torch.randint(-5, far, (T,), generator=g, device=dev).to(pos_dtype)
    return q, k, pos, bsk.rotary_frequencies(r, 500000.0, device=dev)[0]


def _check(got, x, pos, f, inter, scale, sign=1.0):
    # one rounding of the result; the cosine and sine (fp32 fraction of a turn, 2 pi * 2^-25 each, and two roundings each)
    # and the two products' roundings stay below 2^-20 of |a| + |b| <= the row's largest pair
    want = pa.rotary64(x, pos, f, inter, scale, sign)
    r = 2 * f.numel()
    size = x.double()[..., :r].abs().amax(-1, keepdim=True) * 2 * abs(scale)
    bound = pa.half_step(x.dtype) * want.abs() + 2.0 ** -20 * size + pa.tiny(x.dtype)
    assert pa.worst(got, want, bound) <= 1.0
    assert torch.equal(got[..., r:], x[..., r:])  # the rest of the head is copied


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,G,D,r", [(1, 1, 1, 64, 64), (7, 5, 1, 128, 128), (33, 32, 8, 128, 64), (2001, 3, 3, 64, 16),
                                       (5, 2, 1, 80, 80), (3, 2, 2, 96, 20), (9, 4, 2, 256, 256), (4, 1, 1, 6, 2),
                                       (3, 1, 1, 512, 510)])
def test_forward(no_device_error, cuda_dev, dtype, inter, T, H, G, D, r):
    q, k, pos, f = _make(T, H, G, D, r, dtype, cuda_dev)
    for p in (pos, pos.int()):
        qo, ko = bsk.rotary_embedding(q, k, p, f, interleaved=inter, scale=1.2)
        assert qo.is_contiguous() and qo.shape == q.shape and qo.dtype == dtype
        _check(qo, q, pos, f, inter, 1.2)
        _check(ko, k, pos, f, inter, 1.2)
    qo, none = bsk.rotary_embedding(q, None, pos, f, interleaved=inter)
    assert none is None
    _check(qo, q, pos, f, inter, 1.0)


@pytest.mark.parametrize("inter", [False, True])
def test_strided_rows(no_device_error, cuda_dev, inter):
    """Q and K as views of one packed projection, a misaligned view, and a view with another inner stride."""
    T, H, G, D = 19, 6, 2, 64
    x = torch.randn(T, H + 2 * G, D, device=cuda_dev).bfloat16()
    pos, f = torch.arange(T, device=cuda_dev), bsk.rotary_frequencies(D, device=cuda_dev)[0]
    q, k = x[:, :H], x[:, H:H + G]
    qo, ko = bsk.rotary_embedding(q, k, pos, f, interleaved=inter)
    _check(qo, q, pos, f, inter, 1.0)
    _check(ko, k, pos, f, inter, 1.0)
    odd = torch.randn(T * H * D + 1, device=cuda_dev).bfloat16()[1:].view(T, H, D)
    qo, _ = bsk.rotary_embedding(odd, None, pos, f, interleaved=inter)
    _check(qo, odd, pos, f, inter, 1.0)
    turned = torch.randn(T, D, H, device=cuda_dev).bfloat16().transpose(1, 2)
    qo, _ = bsk.rotary_embedding(turned, None, pos[:, None].expand(T, 2)[:, 0], f, interleaved=inter)
    _check(qo, turned, pos, f, inter, 1.0)
    wide = torch.randn(T, 1, D, device=cuda_dev).bfloat16().expand(T, H, D)  # one head, broadcast
    qo, _ = bsk.rotary_embedding(wide, None, pos, f, interleaved=inter)
    _check(qo, wide, pos, f, inter, 1.0)


def test_far_positions(no_device_error, cuda_dev):
    """Positions to 2^40: the angle is exact to a 2^-53 of itself, far below the fp32 rounding that follows."""
    q = torch.randn(64, 2, 128, device=cuda_dev)
    f = bsk.rotary_frequencies(128, device=cuda_dev)[0]
    pos = torch.randint(0, 1 << 27, (64,), device=cuda_dev)
    qo, _ = bsk.rotary_embedding(q, None, pos, f)
    _check(qo, q, pos, f, False, 1.0)


@pytest.mark.parametrize("inter", [False, True])
def test_gradient(no_device_error, cuda_dev, inter):
    q, k, pos, f = _make(37, 4, 2, 64, 32, torch.float32, cuda_dev)
    q.requires_grad_(True)
    k.requires_grad_(True)
    qo, ko = bsk.rotary_embedding(q, k, pos, f, interleaved=inter, scale=0.7)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    _check_grad = lambda got, g: _check(got[..., :32], g[..., :32], pos, f, inter, 0.7, -1.0)  # noqa: E731
    _check_grad(dq, gq)
    _check_grad(dk, gk)
    assert torch.equal(dq[..., 32:], gq[..., 32:])
    # against differences of the (linear) forward: <g, f(x + d) - f(x)> = <grad, d>
    d = torch.randn_like(q)
    with torch.no_grad():
        diff = (gq.double() * (bsk.rotary_embedding(q + d, None, pos, f, interleaved=inter, scale=0.7)[0].double() -
                               qo.double())).sum()
    size = gq.double().norm() * (q.double().norm() + d.double().norm())
    assert abs(diff - (dq.double() * d.double()).sum()) <= 2.0 ** -20 * size
    # one side only
    (only,) = torch.autograd.grad(ko, k, gk, retain_graph=True)
    assert torch.equal(only, dk)
    q2 = q.detach()
    qo2, ko2 = bsk.rotary_embedding(q2, k, pos, f, interleaved=inter, scale=0.7)
    (only,) = torch.autograd.grad((ko2 * gk).sum() + qo2.sum() * 0, k)
    assert torch.equal(only, dk)


def test_refusals(cuda_dev):
    q, k, pos, f = _make(4, 2, 1, 64, 64, torch.float16, cuda_dev)
    bad = [dict(Q=q[0]), dict(Q=q.double()), dict(Q=q.cpu()), dict(K=k[:2]), dict(K=k.float()), dict(K=k[..., :32]),
           dict(positions=pos[:3]), dict(positions=pos.float()), dict(positions=pos.cpu()), dict(inv_freq=f.double()),
           dict(inv_freq=torch.ones(33, device=cuda_dev)), dict(inv_freq=f[:0]), dict(Q=q[..., :63], K=None, inv_freq=f[:4])]
    for change in bad:
        args = dict(Q=q, K=k, positions=pos, inv_freq=f)
        args.update(change)
        with pytest.raises(ValueError):
            bsk.rotary_embedding(**args)
    with pytest.raises(ValueError, match="inv_freq"):
        bsk.rotary_embedding(q, k, pos, f.clone().requires_grad_(True))
    qo, ko = bsk.rotary_embedding(q[:0], k[:0], pos[:0], f)  # no tokens is no error
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 1, 64)
