"""Norm of each head with the rotation, forward and gradients, against the 64-bit definition within its roundings: layouts, types
of rows and weights, head sizes that take each of the kernel's vector widths, strides, zero and huge rows, several axes,
streams, graphs, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu
EPS = 1e-6


def make(T, H, G, D, dtype, dev, wdtype=None, seed=0, size=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, k, dq, dk = (torch.randn(T, n, D, generator=g, device=dev).to(dtype) for n in (H, G, H, G))
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(wdtype or dtype) for _ in range(2))
    pos = torch.randint(-5, 100000, (T,), generator=g, device=dev)
    return q * size, k * size, qw, kw, dq, dk, pos


def grads(q, k, qw, kw, dq, dk, pos, f, **kw_args):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    qo, ko = bsk.qk_norm_rotary(*leaves, pos, f, **kw_args)
    return (qo.detach(), ko.detach(), *torch.autograd.grad((qo, ko), leaves, (dq, dk)))


def check(got, q, k, qw, kw, dq, dk, pos, f, interleaved=False, scale=1.0, eps=EPS, axes=None):
    qo, ko, gq, gk, gqw, gkw = got
    for x, w, dy, y, dx, dw in ((q, qw, dq, qo, gq, gqw), (k, kw, dk, ko, gk, gkw)):
        want = pa.norm_rotary64(x, w, pos, f, interleaved, scale, eps, axes, dy)
        for name, t in (("y", y), ("dx", dx), ("dw", dw)):
            assert t.shape == want[name][0].shape and t.dtype == (w.dtype if name == "dw" else x.dtype)
            r = pa.worst(t, *want[name])
            assert r <= 1.0, (name, r)


SHAPES = [  # tokens, heads, kv heads, dim, turned elements
    (1, 1, 1, 64, 64), (7, 5, 1, 128, 128), (33, 32, 8, 128, 64), (2001, 3, 3, 64, 16), (5, 2, 1, 80, 80), (300, 4, 2, 80, 40),
    (3, 2, 2, 96, 20), (9, 4, 2, 256, 256), (4, 1, 1, 6, 2), (3, 1, 1, 512, 510), (70, 40, 1, 512, 512), (1300, 12, 4, 96, 96),
    (700, 1, 1, 192, 96), (611, 128, 2, 16, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,G,D,r", SHAPES)
def test_against_definition(no_device_error, cuda_dev, dtype, inter, T, H, G, D, r):
    f = bsk.rotary_frequencies(r, 500000.0, device=cuda_dev)[0]
    for wdtype in {dtype, torch.float32}:
        x = make(T, H, G, D, dtype, cuda_dev, wdtype, seed=T + D)
        got = grads(*x, f, interleaved=inter, scale=1.2)
        check(got, *x, f, inter, 1.2)
        again = grads(*x, f, interleaved=inter, scale=1.2)
        assert all(torch.equal(a, b) for a, b in zip(again, got))  # deterministic
        with torch.no_grad():
            alone, none = bsk.qk_norm_rotary(x[0], None, x[2], None, x[6].int(), f, interleaved=inter, scale=1.2)
        assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_of_every_size(no_device_error, cuda_dev, dtype):
    """Rows of zeros, tiny rows (eps decides) and, but for fp16, rows whose squares pass fp32's range."""
    f = bsk.rotary_frequencies(128, device=cuda_dev)[0]
    x = list(make(200, 4, 2, 128, dtype, cuda_dev))
    sizes = [0.0, 1e-4, 1.0, 100.0] + ([1e19, 1e30, 5e37] if dtype != torch.float16 else [1e4])
    for i in (0, 1):
        for j, size in enumerate(sizes):
            x[i][j::len(sizes)] = (x[i][j::len(sizes)].float().clamp(-4, 4) * size).to(dtype)
    got = grads(*x, f)
    assert all(torch.isfinite(t).all() for t in got)
    check(got, *x, f)
    assert (got[0][0] == 0).all()


@pytest.mark.parametrize("T,H,G,D,r", [(593, 1, 64, 64, 64), (593, 64, 1, 64, 32), (20000, 2, 1, 6, 4), (4097, 16, 16, 96, 96),
                                       (1777, 1, 1, 512, 512), (2500, 33, 7, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_heads_and_tokens_of_many_proportions(no_device_error, cuda_dev, dtype, T, H, G, D, r):
    """How heads and tokens are dealt to blocks follows the costs of Q and K: few heads beside many, odd ones, alone."""
    f = bsk.rotary_frequencies(r, device=cuda_dev)[0]
    x = make(T, H, G, D, dtype, cuda_dev, torch.float32, seed=H + G)
    got = grads(*x, f)
    check(got, *x, f)
    for i, j in ((0, 2), (1, 3)):  # each alone is dealt in another way
        with torch.no_grad():
            assert torch.equal(bsk.qk_norm_rotary(x[i], None, x[j], None, x[6], f)[0], got[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
def test_large_rows_and_a_large_scale(no_device_error, cuda_dev, dtype, inter):
    """Rows of 1e18 times a scale of 1e25 pass fp32's range, their results do not."""
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    q, k, qw, kw, _, _, pos = make(50, 4, 2, 128, dtype, cuda_dev, size=1e18)
    for x, w, y in zip((q, k), (qw, kw), bsk.qk_norm_rotary(q, k, qw, kw, pos, f, interleaved=inter, scale=1e25)):
        assert torch.isfinite(y).all()
        assert pa.worst(y, *pa.norm_rotary64(x, w, pos, f, inter, 1e25, EPS)["y"]) <= 1.0


@pytest.mark.parametrize("eps", [1e-30, 1e-3, 10.0])
def test_eps(no_device_error, cuda_dev, eps):
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = make(50, 3, 1, 64, torch.float32, cuda_dev, size=0.1)
    check(grads(*x, f, eps=eps), *x, f, eps=eps)


def test_non_finite_rows_stay_by_themselves(no_device_error, cuda_dev):
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = list(make(50, 4, 2, 64, torch.bfloat16, cuda_dev))
    want = grads(*x, f)
    x[0] = x[0].clone()
    x[0][3, 1, 5], x[0][20, 2, 60] = float("nan"), float("inf")
    got = grads(*x, f)
    rows = torch.ones(50, 4, dtype=torch.bool, device=cuda_dev)
    rows[3, 1] = rows[20, 2] = False
    for i in (0, 2):
        assert torch.equal(got[i][rows], want[i][rows])
    assert torch.isnan(got[0][3, 1]).all() and torch.isnan(got[0][20, 2, 60])
    assert all(torch.equal(got[i], want[i]) for i in (1, 3, 5))


@pytest.mark.parametrize("inter", [False, True])
def test_strided_rows(no_device_error, cuda_dev, inter):
    """Q and K as views of one packed projection, a misaligned view, another inner stride, a broadcast head, broadcast gradients
    and weights that are views."""
    T, H, G, D = 19, 6, 2, 64
    f = bsk.rotary_frequencies(D, device=cuda_dev)[0]
    x = list(make(T, H, G, D, torch.bfloat16, cuda_dev))
    want = grads(*x, f, interleaved=inter)
    packed = torch.cat([x[0], x[1], x[1]], 1)
    odd = torch.empty(x[0].numel() + 1, dtype=x[0].dtype, device=cuda_dev)[1:].view_as(x[0]).copy_(x[0])
    inner = x[0].transpose(1, 2).contiguous().transpose(1, 2)
    weights = torch.stack([x[2], x[3]], 1)
    for q in (packed[:, :H], odd, inner):
        got = grads(q, packed[:, H:H + G], weights[:, 0], weights[:, 1], *x[4:], f, interleaved=inter)
        check(got, *x, f, inter)
        if q is not odd:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    x[0] = x[0][:, :1].expand(T, H, D)
    x[4] = x[4][:, :, :1].expand(T, H, D)
    check(grads(*x, f, interleaved=inter), *x, f, inter)


def test_several_axes(no_device_error, cuda_dev):
    f = bsk.rotary_frequencies(128, device=cuda_dev)[0]
    x = list(make(300, 8, 2, 128, torch.bfloat16, cuda_dev))
    for sections, cycle in (((16, 24, 24), False), ((24, 20, 20), True)):
        axes = bsk.rotary_axes(sections, cycle, device=cuda_dev)
        x[6] = torch.randint(0, 5000, (3, 300), device=cuda_dev)
        check(grads(*x, f, axes=axes), *x, f, axes=axes)


def test_gradients_of_some_inputs_only(no_device_error, cuda_dev):
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    q, k, qw, kw, dq, dk, pos = make(40, 4, 2, 64, torch.bfloat16, cuda_dev)
    want = grads(q, k, qw, kw, dq, dk, pos, f)
    for pick in range(4):
        leaves = [t.detach().requires_grad_(i == pick) for i, t in enumerate((q, k, qw, kw))]
        qo, ko = bsk.qk_norm_rotary(*leaves, pos, f)
        (g,) = torch.autograd.grad((qo, ko)[pick % 2], leaves[pick], (dq, dk)[pick % 2])
        assert torch.equal(g, want[2 + pick])
    leaf = q.detach().requires_grad_(True)
    qo, _ = bsk.qk_norm_rotary(leaf, None, qw, None, pos, f)
    assert torch.equal(torch.autograd.grad(qo, leaf, dq)[0], want[2])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    qo, ko = bsk.qk_norm_rotary(*leaves, pos, f)
    (g,) = torch.autograd.grad(qo.sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        g.sum().backward()


def test_gradient_against_differences(no_device_error, cuda_dev):
    """<dy, y(x + h d) - y(x - h d)> / 2h in 64 bits against the kernel's <gradient, d>: the gradient's bound, and the
    differences' h^2 term (third derivatives of a row's norm stay below 100 / rms^3 here)."""
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = make(20, 3, 1, 64, torch.float32, cuda_dev)
    got = grads(*x, f)
    h = 1e-5
    for i, name in ((0, "dx"), (2, "dw")):
        want = pa.norm_rotary64(x[0], x[2], x[6], f, False, 1.0, EPS, None, x[4])[name]
        d = torch.randn_like(x[i].double())
        ends = []
        for s in (h, -h):
            a = [x[0].double(), x[2].double()]
            a[i // 2] = a[i // 2] + s * d
            ends.append((_forward64(*a, x[6], f) * x[4].double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        assert abs(slope - (got[2 + i].double() * d).sum()) <= (want[1] * d.abs()).sum() + 1e-6 * x[4].double().norm()


def _forward64(x, w, pos, f):
    unit = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    return pa.rotary64(unit * w, pos, f, False, 1.0)


def test_another_stream_and_captured_steps(no_device_error, cuda_dev):
    f = bsk.rotary_frequencies(128, device=cuda_dev)[0]
    x = make(900, 8, 2, 128, torch.bfloat16, cuda_dev)
    want = grads(*x, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grads(*x, f)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.detach().clone().requires_grad_(True) for t in x[:4]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = bsk.qk_norm_rotary(*leaves, x[6], f)
        out = (*(t.detach() for t in o), *torch.autograd.grad(o, leaves, (x[4], x[5])))
        del o
    with torch.no_grad():
        leaves[0].copy_(x[0].flip(0))
        leaves[2].copy_(x[2].flip(0))
    graph.replay()
    want = grads(x[0].flip(0), x[1], x[2].flip(0), *x[3:], f)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_no_tokens_and_refusals(cuda_dev):
    f = bsk.rotary_frequencies(64, device=cuda_dev)[0]
    x = make(4, 2, 1, 64, torch.float16, cuda_dev)
    empty = grads(*(t[:0] for t in x[:2]), *x[2:4], *(t[:0] for t in x[4:]), f)
    assert empty[0].shape == (0, 2, 64) and empty[3].shape == (0, 1, 64) and (empty[4] == 0).all() and (empty[5] == 0).all()
    q, k, qw, kw, _, _, pos = x
    good = dict(Q=q, K=k, q_weight=qw, k_weight=kw, positions=pos, inv_freq=f)
    bsk.qk_norm_rotary(**good)
    for change in (dict(Q=q[0]), dict(Q=q.double()), dict(Q=q.cpu()), dict(K=k[:2]), dict(K=k.float()), dict(K=None), dict(k_weight=None),
                   dict(q_weight=qw[:63]), dict(q_weight=qw.bfloat16()), dict(q_weight=qw.cpu()), dict(q_weight=qw.float()),
                   dict(q_weight=qw[None]), dict(positions=pos[:3]), dict(inv_freq=f.double()), dict(eps=0.0), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("inf")), dict(inv_freq=f.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            bsk.qk_norm_rotary(**{**good, **change})
    import torch.autograd.forward_ad as fwd

    for n in ("Q", "K", "q_weight", "k_weight"):
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            bsk.qk_norm_rotary(**{**good, n: fwd.make_dual(good[n], torch.ones_like(good[n]))})
