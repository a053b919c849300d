"""Norm with rotation of Q alone (K and its weight absent): every set of inputs that require a gradient gets what it gets beside
K, within the definition's roundings."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from test_gpu_norm_rotary import EPS, grads, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("several_axes", [False, True])
@pytest.mark.parametrize("T", [1, 40, 2500])  # few tokens and many are dealt to blocks in two ways
def test_gradients_without_k(no_device_error, cuda_dev, T, several_axes, dtype, wdtype):
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = list(make(T, 6, 2, 64, dtype, cuda_dev, wdtype, seed=T))
    axes = bsk.rotary_axes((12, 10, 10), device=cuda_dev) if several_axes else None
    if several_axes:
        x[6] = torch.randint(0, 5000, (3, T), device=cuda_dev)
    q, _, qw, _, dq, _, pos = x
    beside = grads(*x, f, axes=axes)
    want = pa.norm_rotary64(q, qw, pos, f, False, 1.0, EPS, axes, dq)
    for need_q, need_w in ((True, False), (False, True), (True, True)):
        leaf, weight = q.detach().requires_grad_(need_q), qw.detach().requires_grad_(need_w)
        out, none = bsk.qk_norm_rotary(leaf, None, weight, None, pos, f, axes=axes)
        assert none is None and torch.equal(out, beside[0])
        out.backward(dq)
        assert (leaf.grad is not None) == need_q and (weight.grad is not None) == need_w
        if need_q:
            assert torch.equal(leaf.grad, beside[2])
        if need_w:
            assert weight.grad.dtype == wdtype and pa.worst(weight.grad, *want["dw"]) <= 1.0


def test_one_result_of_two(no_device_error, cuda_dev):
    """A loss over one result of a call with both gives the other's inputs no gradient, and a weight that both share gets its sum."""
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = make(40, 4, 2, 64, torch.bfloat16, cuda_dev, torch.float32)
    want = grads(*x, f)
    for i in (0, 1):
        leaves = [t.detach().requires_grad_(True) for t in x[:4]]
        bsk.qk_norm_rotary(*leaves, x[6], f)[i].backward(x[4 + i])
        assert torch.equal(leaves[i].grad, want[2 + i]) and torch.equal(leaves[2 + i].grad, want[4 + i])
        assert leaves[1 - i].grad is None and leaves[3 - i].grad is None
    w = x[2].detach().requires_grad_(True)
    qo, ko = bsk.qk_norm_rotary(x[0], x[1], w, w, x[6], f)
    torch.autograd.backward((qo, ko), (x[4], x[5]))
    dk = pa.norm_rotary64(x[1], x[2], x[6], f, False, 1.0, EPS, None, x[5])["dw"]
    dq = pa.norm_rotary64(x[0], x[2], x[6], f, False, 1.0, EPS, None, x[4])["dw"]
    total = dq[0] + dk[0]
    assert pa.worst(w.grad, total, dq[1] + dk[1] + 2.0 ** -24 * total.abs()) <= 1.0
