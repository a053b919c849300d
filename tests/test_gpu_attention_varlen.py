"""Attention over packed sequences, forward and gradients, against the 64-bit definition, elementwise within the
roundings' bound: lengths from one token on, odd sizes, group sizes, types, strides, neighbours full of NaN, streams,
graphs, bad indices, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def make(lens, H, G, D, dtype, dev, seed=0, size=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lens)
    q, do = (torch.randn(T, H, D, generator=g, device=dev).mul(s).to(dtype) for s in (size, 1.0))
    k, v = (torch.randn(T, G, D, generator=g, device=dev).to(dtype) for _ in range(2))
    return q, k, v, do, torch.tensor([0] + lens, device=dev).cumsum(0).int()


def grads(q, k, v, do, cu, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = bsk.attention_varlen(q, k, v, cu, **kw)
    return dict(zip(("O", "dQ", "dK", "dV"), (o.detach(), *torch.autograd.grad(o, (q, k, v), do))))


def check(got, q, k, v, do, lens, causal, scale=None):
    want = pa.packed64(q, k, v, lens, causal, scale or q.shape[2] ** -0.5, do)
    for name, (val, bound) in want.items():
        assert got[name].dtype == q.dtype and got[name].shape == val.shape
        w = pa.worst(got[name], val, bound)
        assert w <= 1.0, (name, w)


SHAPES = [  # lengths, heads, kv heads
    ([1], 1, 1), ([1, 1, 2], 4, 2), ([128], 2, 2), ([127, 129], 2, 1), ([5, 0, 300, 0], 8, 2), ([64, 65, 63, 1, 200], 6, 2),
    ([257, 512, 31], 5, 1), ([1000], 8, 8), ([700, 33], 3, 3), ([40] * 12, 7, 1), ([90, 130], 128, 1), ([513], 16, 1),
    ([2049, 3], 2, 2),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G", SHAPES)
def test_against_definition(no_device_error, cuda_dev, lens, H, G, D, dtype, causal):
    q, k, v, do, cu = make(lens, H, G, D, dtype, cuda_dev, seed=H + D)
    got = grads(q, k, v, do, cu, causal=causal)
    check(got, q, k, v, do, lens, causal)
    assert torch.equal(bsk.attention_varlen(q, k, v, cu.long(), causal=causal), got["O"])  # without a gradient
    again = grads(q, k, v, do, cu, causal=causal)
    assert all(torch.equal(again[n], got[n]) for n in got)  # deterministic


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_and_scale(no_device_error, cuda_dev, dtype):
    q, k, v, do, cu = make([300, 77], 4, 2, 64, dtype, cuda_dev, size=6.0)
    check(grads(q, k, v, do, cu, scale=0.3), q, k, v, do, [300, 77], True, 0.3)


def test_neighbours_do_not_reach_in(no_device_error, cuda_dev):
    """A sequence between two full of NaN and infinities gets exactly the values it gets between ordinary ones."""
    lens = [77, 203, 60]
    for H, G, D in ((4, 2, 128), (6, 1, 64)):
        q, k, v, do, cu = make(lens, H, G, D, torch.bfloat16, cuda_dev)
        want = grads(q, k, v, do, cu)
        for t, x in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (do, float("-inf"))):
            t[:77], t[280:] = x, x
        got = grads(q, k, v, do, cu)
        for n in got:
            assert torch.equal(got[n][77:280], want[n][77:280]), n


def test_non_finite_values_reach_the_rows_that_see_them_only(no_device_error, cuda_dev):
    """A NaN key is seen by itself and later rows; a NaN query row by itself, its dQ and (through dK, dV) all keys it sees."""
    q, k, v, do, cu = make([300], 4, 2, 64, torch.bfloat16, cuda_dev)
    want = grads(q, k, v, do, cu)
    k2 = k.clone()
    k2[200, 1, 3] = float("nan")
    got = grads(q, k2, v, do, cu)
    assert torch.equal(got["O"][:200], want["O"][:200]) and torch.equal(got["O"][200:, :2], want["O"][200:, :2])
    assert torch.isnan(got["O"][200:, 2:]).all() and torch.isnan(got["dQ"][200:, 2:]).all()
    q2 = q.clone()
    q2[100, 0, 5] = float("inf")
    got = grads(q2, k, v, do, cu)
    rows = torch.ones(300, 4, dtype=torch.bool, device=cuda_dev)
    rows[100, 0] = False
    for n in ("O", "dQ"):
        assert torch.equal(got[n][rows], want[n][rows]) and torch.isnan(got[n][100, 0]).all()
    assert torch.equal(got["dK"][:, 1], want["dK"][:, 1]) and torch.isnan(got["dK"][:101, 0]).any(-1).all()
    assert torch.equal(got["dK"][128:, 0], want["dK"][128:, 0])  # keys behind the row's last block


def test_rows_behind_the_last_sequence_are_zero(no_device_error, cuda_dev):
    q, k, v, do, cu = make([100, 30, 171], 4, 2, 64, torch.float16, cuda_dev)
    want = grads(q[:130], k[:130], v[:130], do[:130], cu[:3])
    for t in (q, k, v, do):
        t[130:] = float("nan")
    got = grads(q, k, v, do, cu[:3])
    for n in got:
        assert torch.equal(got[n][:130], want[n]) and (got[n][130:] == 0).all(), n
    none = grads(q, k, v, do, cu[:1])
    assert all((none[n] == 0).all() for n in none)
    empty = grads(q[:0], k[:0], v[:0], do[:0], cu[:1])
    assert empty["O"].shape == (0, 4, 64) and empty["dK"].shape == (0, 2, 64)


def test_strides_and_broadcast_gradients(no_device_error, cuda_dev):
    lens, H, G, D = [150, 61], 4, 2, 64
    q, k, v, do, cu = make(lens, H, G, D, torch.bfloat16, cuda_dev)
    want = grads(q, k, v, do, cu)
    qkv = torch.cat([q, k, v], 1)
    views = (qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:])
    got = grads(*views, do.transpose(0, 1).contiguous().transpose(0, 1), cu)
    assert all(torch.equal(got[n], want[n]) for n in got)
    got = grads(*views, do[:, :1, :1].expand_as(do), cu)  # a gradient that is one value broadcast
    check(got, q, k, v, do[:, :1, :1].expand_as(do).contiguous(), lens, True)
    # one packed leaf: the three gradients land in its parts
    leaf = qkv.detach().requires_grad_(True)
    o = bsk.attention_varlen(leaf[:, :H], leaf[:, H:H + G], leaf[:, H + G:], cu)
    (g,) = torch.autograd.grad(o, leaf, do)
    assert torch.equal(g, torch.cat([want["dQ"], want["dK"], want["dV"]], 1))
    # gradients asked for one input only
    kk = k.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(bsk.attention_varlen(q, kk, v, cu), kk, do)
    assert torch.equal(g, want["dK"])


def test_gradient_against_differences(no_device_error, cuda_dev):
    """<dO, O(x + h d) - O(x - h d)> / 2h in the oracle's 64 bits against the kernel's <gradient, d>: the gradient's own
    bound, plus the differences' h^2 term."""
    lens = [70, 35]
    q, k, v, do, cu = make(lens, 4, 2, 64, torch.float16, cuda_dev)
    got, bounds = grads(q, k, v, do, cu), pa.packed64(q, k, v, lens, True, 0.125, do)
    h = 1e-4
    for i, name in enumerate(("dQ", "dK", "dV")):
        d = torch.randn_like((q, k, v)[i].double())
        at = [q.double(), k.double(), v.double()]
        ends = []
        for s in (h, -h):
            x = list(at)
            x[i] = at[i] + s * d
            ends.append((pa.packed64(x[0], x[1], x[2], lens, True, 0.125)["O"][0] * do.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        allowed = (bounds[name][1] * d.abs()).sum() + 1e-4 * do.double().norm()
        assert abs(slope - (got[name].double() * d).sum()) <= allowed


def test_another_stream_and_captured_steps(no_device_error, cuda_dev):
    lens = [130, 60]
    q, k, v, do, cu = make(lens, 4, 2, 128, torch.bfloat16, cuda_dev)
    want = grads(q, k, v, do, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = grads(q, k, v, do, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(other[n], want[n]) for n in want)
    # forward and backward captured, twice, in one pool. (No eager graph of the same leaves may live meanwhile: torch ties a
    # leaf's gradient node to the stream of its first use, and a capture that waits for another stream is invalid.)
    ql, kl, vl = (t.detach().clone().requires_grad_(True) for t in (q, k, v))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=graphs[0][0].pool() if graphs else None):
            o = bsk.attention_varlen(ql, kl, vl, cu)
            out = (o.detach(), *torch.autograd.grad(o, (ql, kl, vl), do))
        graphs.append((gr, out))
    for step in range(2):
        with torch.no_grad():
            ql.copy_(torch.randn_like(ql))
        want = grads(ql, kl, vl, do, cu)  # (on detached leaves)
        for gr, out in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, want[n]) for a, n in zip(out, ("O", "dQ", "dK", "dV")))


def test_second_derivatives_are_refused(no_device_error, cuda_dev):
    q, k, v, do, cu = make([20, 9], 2, 1, 64, torch.float16, cuda_dev)
    q.requires_grad_(True)
    (g,) = torch.autograd.grad(bsk.attention_varlen(q, k, v, cu), q, do, create_graph=True)
    assert torch.equal(g.detach(), grads(q, k, v, do, cu)["dQ"])
    with pytest.raises(RuntimeError, match="twice differentiable"):
        g.float().sum().backward()
    pos, f = torch.arange(29, device=cuda_dev), bsk.rotary_frequencies(64, device=cuda_dev)[0]
    (g,) = torch.autograd.grad(bsk.rotary_embedding(q, None, pos, f)[0], q, do, create_graph=True)
    with pytest.raises(RuntimeError, match="twice differentiable"):
        g.float().sum().backward()


def test_bad_lengths_are_reported_not_followed(cuda_dev):
    assert _capi.device_error() == 0
    q, k, v, do, cu = make([100, 60], 4, 2, 64, torch.bfloat16, cuda_dev)
    for bad in ([0, 100, 165], [0, 100, 90], [0, -5, 160], [7, 100, 160], [0, 2 ** 31 - 1, 160]):
        grads(q, k, v, do, torch.tensor(bad, dtype=torch.int32, device=cuda_dev))
        with pytest.raises(RuntimeError, match="out-of-range"):
            bsk.synchronize_and_check()
    check(grads(q, k, v, do, cu), q, k, v, do, [100, 60], True)
    assert _capi.device_error() == 0


def test_refusals(cuda_dev):
    q, k, v, do, cu = make([10, 6], 4, 2, 64, torch.bfloat16, cuda_dev)
    base = dict(Q=q, K=k, V=v, cu_seqlens=cu)
    bad = [dict(Q=q[0]), dict(Q=q.float(), K=k.float(), V=v.float()), dict(Q=q.half()), dict(V=v.half()), dict(Q=q.cpu()),
           dict(K=k[:5]), dict(V=v[:5]), dict(K=k[:, :1]), dict(Q=q[:, :3]), dict(Q=q[..., :32], K=k[..., :32], V=v[..., :32]),
           dict(cu_seqlens=cu.float()), dict(cu_seqlens=cu.cpu()), dict(cu_seqlens=cu[None]), dict(cu_seqlens=cu[:0]),
           dict(scale=0.0), dict(scale=float("inf")), dict(Q=q[:, :0])]
    for change in bad:
        with pytest.raises(ValueError):
            bsk.attention_varlen(**{**base, **change})
    wide = torch.zeros(4, 129, 64, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(ValueError, match="128"):
        bsk.attention_varlen(wide, k[:4, :1], v[:4, :1], cu[:1])
