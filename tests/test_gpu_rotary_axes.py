"""Rotary positions with several axes against their 64-bit definition: runs and turns of the axes, layouts, types, partial heads,
gradients, one axis, axes out of range, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def check(got, x, pos, f, inter, scale, axes, sign=1.0):
    want = pa.rotary64(x, pos, f, inter, scale, sign, axes)
    r = 2 * f.numel()
    size = x.double()[..., :r].abs().amax(-1, keepdim=True) * 2 * abs(scale)
    bound = pa.half_step(x.dtype) * want.abs() + pa.TURN * size + pa.tiny(x.dtype)
    assert pa.worst(got, want, bound) <= 1.0
    assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("cycle", [False, True])
@pytest.mark.parametrize("T,H,G,D,sections", [(1, 1, 1, 64, (16, 16)), (33, 32, 8, 128, (16, 24, 24)), (700, 3, 3, 128, (24, 20, 20)),
                                              (5, 2, 1, 80, (0, 13, 27)), (2001, 4, 2, 64, (8,)), (9, 2, 2, 96, (1, 2, 3, 4)),
                                              (4, 1, 1, 6, (0, 1, 0))])
def test_forward_and_gradient(no_device_error, cuda_dev, dtype, inter, cycle, T, H, G, D, sections):
    g = torch.Generator(device=cuda_dev).manual_seed(T + D)
    q, k = (torch.randn(T, n, D, generator=g, device=cuda_dev).to(dtype) for n in (H, G))
    axes = bsk.rotary_axes(sections, cycle, device=cuda_dev)
    f = bsk.rotary_frequencies(2 * sum(sections), 500000.0, device=cuda_dev)[0]
    pos = torch.randint(-5, 100000, (len(sections), T), generator=g, device=cuda_dev)
    q, k = q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = bsk.rotary_embedding(q, k, pos, f, interleaved=inter, scale=1.2, axes=axes)
    check(qo.detach(), q.detach(), pos, f, inter, 1.2, axes)
    check(ko.detach(), k.detach(), pos, f, inter, 1.2, axes)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    r = 2 * f.numel()
    check(dq[..., :r], gq[..., :r], pos, f, inter, 1.2, axes, -1.0)
    check(dk[..., :r], gk[..., :r], pos, f, inter, 1.2, axes, -1.0)
    assert torch.equal(dq[..., r:], gq[..., r:])
    with torch.no_grad():
        again, none = bsk.rotary_embedding(q, None, pos.int(), f, interleaved=inter, scale=1.2, axes=axes.long())
    assert none is None and torch.equal(again, qo)


def test_axes_that_agree_are_one_axis(no_device_error, cuda_dev):
    """Text tokens have one position on all axes: bit for bit the plain rotation."""
    q = torch.randn(50, 4, 128, device=cuda_dev).bfloat16()
    k = torch.randn(50, 2, 128, device=cuda_dev).bfloat16()
    f = bsk.rotary_frequencies(128, device=cuda_dev)[0]
    pos = torch.arange(1000, 1050, device=cuda_dev)
    want = bsk.rotary_embedding(q, k, pos, f)
    for sections, cycle in (((16, 24, 24), False), ((24, 20, 20), True), ((64,), False)):
        axes = bsk.rotary_axes(sections, cycle, device=cuda_dev)
        got = bsk.rotary_embedding(q, k, pos.expand(len(sections), 50), f, axes=axes)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_axes_out_of_range_are_reported(cuda_dev):
    q = torch.randn(5, 1, 64, device=cuda_dev)
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    pos = torch.randint(0, 99, (2, 5), device=cuda_dev)
    axes = torch.arange(32, device=cuda_dev) % 4 - 1
    assert _capi.device_error() == 0
    got = bsk.rotary_embedding(q, None, pos, f, axes=axes)[0]
    with pytest.raises(RuntimeError):
        bsk.synchronize_and_check()
    assert torch.equal(got, bsk.rotary_embedding(q, None, pos, f, axes=axes.clamp(0, 1))[0])
    bsk.synchronize_and_check()


def test_refusals(cuda_dev):
    q = torch.randn(4, 2, 64, device=cuda_dev)
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    pos, axes = torch.zeros(3, 4, dtype=torch.int64, device=cuda_dev), bsk.rotary_axes((10, 11, 11), device=cuda_dev)
    bsk.rotary_embedding(q, None, pos, f, axes=axes)
    for kw in (dict(positions=pos[0]), dict(positions=pos[:, :3]), dict(positions=pos[:0]), dict(axes=axes[:31]), dict(axes=axes.float()),
               dict(axes=axes.cpu()), dict(axes=axes[None]), dict(axes=None)):
        with pytest.raises(ValueError):
            bsk.rotary_embedding(q, None, **{**dict(positions=pos, inv_freq=f, axes=axes), **kw})
