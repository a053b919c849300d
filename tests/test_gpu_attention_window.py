"""Packed attention with a sliding window and sinks, forward and gradients, against the 64-bit definition, elementwise within
the roundings' bound: windows from one token to longer than the sequences, sinks inside and across key blocks, group sizes,
lengths around the tiles' ends, values that a row does not see, streams, graphs, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from test_gpu_attention_varlen import grads, make

pytestmark = pytest.mark.gpu


def check(got, q, k, v, do, lens, window, sinks, scale=None):
    want = pa.packed64(q, k, v, lens, True, scale or q.shape[2] ** -0.5, do, window, sinks)
    for name, (val, bound) in want.items():
        assert got[name].dtype == q.dtype and got[name].shape == val.shape
        w = pa.worst(got[name], val, bound)
        assert w <= 1.0, (name, w)


SHAPES = [  # lengths, heads, kv heads, window, sinks
    ([1, 1], 1, 1, 1, 0), ([300], 2, 2, 1, 0), ([300], 4, 2, 1, 1), ([5, 0, 300, 0], 8, 2, 7, 3), ([257, 512, 31], 5, 1, 64, 0),
    ([700, 33], 3, 3, 100, 4), ([640], 2, 1, 128, 0), ([640], 2, 1, 129, 128), ([900, 130], 8, 2, 127, 130), ([90, 430], 128, 1, 50, 2),
    ([1000], 8, 8, 300, 0), ([40] * 12, 7, 1, 33, 5), ([2049, 3], 2, 2, 700, 260), ([513], 16, 1, 256, 1), ([1300], 4, 4, 31, 500),
    ([200, 77], 4, 2, 200, 9), ([127, 129], 2, 1, 4096, 4),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G,window,sinks", SHAPES)
def test_against_definition(no_device_error, cuda_dev, lens, H, G, D, dtype, window, sinks):
    q, k, v, do, cu = make(lens, H, G, D, dtype, cuda_dev, seed=H + D + window)
    got = grads(q, k, v, do, cu, window=window, sinks=sinks)
    check(got, q, k, v, do, lens, window, sinks)
    assert torch.equal(bsk.attention_varlen(q, k, v, cu.long(), window=window, sinks=sinks), got["O"])  # without a gradient
    again = grads(q, k, v, do, cu, window=window, sinks=sinks)
    assert all(torch.equal(again[n], got[n]) for n in got)  # deterministic


@pytest.mark.parametrize("window,sinks", [(300, 0), (10 ** 6, 3), (1, 299), (150, 150), (2 ** 40, 2 ** 40)])
def test_windows_that_leave_nothing_out(no_device_error, cuda_dev, window, sinks):
    """The results are those of plain causal attention, bit for bit."""
    q, k, v, do, cu = make([300, 77], 4, 2, 64, torch.bfloat16, cuda_dev)
    want = grads(q, k, v, do, cu)
    if window + sinks >= 377:  # (known from the tensors' sizes: the same kernels)
        got = grads(q, k, v, do, cu, window=window, sinks=sinks)
        assert all(torch.equal(got[n], want[n]) for n in got)
    else:
        check(grads(q, k, v, do, cu, window=window, sinks=sinks), q, k, v, do, [300, 77], window, sinks)
        check(want, q, k, v, do, [300, 77], window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_and_scale(no_device_error, cuda_dev, dtype):
    q, k, v, do, cu = make([500, 77], 4, 2, 64, dtype, cuda_dev, size=6.0)
    check(grads(q, k, v, do, cu, scale=0.3, window=90, sinks=2), q, k, v, do, [500, 77], 90, 2, 0.3)


def test_keys_behind_the_window_reach_nothing(no_device_error, cuda_dev):
    """Large finite keys and values that rows do not see change no bit of their results; nor do NaN keys of O, dK and dV. A NaN
    value meets a weight of zero in O, a NaN key a zero of dS in dQ, of rows fewer than 256 tokens from those that see it."""
    q, k, v, do, cu = make([900], 4, 2, 64, torch.bfloat16, cuda_dev)
    kw = dict(window=100, sinks=3)
    want = grads(q, k, v, do, cu, **kw)
    k2, v2 = k.clone(), v.clone()
    k2[200], v2[200] = 3e38, 3e38
    got = grads(q, k2, v2, do, cu, **kw)
    rows = torch.ones(900, dtype=torch.bool, device=cuda_dev)
    rows[200:300] = False
    for n in ("O", "dQ"):
        assert torch.equal(got[n][rows], want[n][rows]), n
    k2[200], v2[200] = float("nan"), v[200]
    got = grads(q, k2, v2, do, cu, **kw)
    assert torch.equal(got["O"][rows], want["O"][rows]) and torch.equal(got["dQ"][556:], want["dQ"][556:])
    assert torch.isnan(got["O"][200:300]).all() and torch.isnan(got["dQ"][200:300]).all()
    keys = torch.ones(900, dtype=torch.bool, device=cuda_dev)
    keys[101:300] = False  # seen by rows 200 .. 299, as are the sinks
    keys[:3] = False
    for n in ("dK", "dV"):
        assert torch.equal(got[n][keys], want[n][keys]), n
    v2[200], k2[200] = float("nan"), k[200]
    got = grads(q, k2, v2, do, cu, **kw)
    assert torch.equal(got["O"][556:], want["O"][556:]) and torch.isnan(got["O"][200:300]).all()


def test_rows_without_a_gradient_and_rows_behind_the_last_sequence(no_device_error, cuda_dev):
    q, k, v, do, cu = make([400, 30, 171], 4, 2, 64, torch.float16, cuda_dev)
    kw = dict(window=60, sinks=1)
    want = grads(q[:430], k[:430], v[:430], do[:430], cu[:3], **kw)
    for t in (q, k, v, do):
        t[430:] = float("nan")
    got = grads(q, k, v, do, cu[:3], **kw)
    for n in got:
        assert torch.equal(got[n][:430], want[n]) and (got[n][430:] == 0).all(), n
    empty = grads(q[:0], k[:0], v[:0], do[:0], cu[:1], **kw)
    assert empty["O"].shape == (0, 4, 64) and empty["dK"].shape == (0, 2, 64)


def test_gradient_against_differences(no_device_error, cuda_dev):
    """<dO, O(x + h d) - O(x - h d)> / 2h in the oracle's 64 bits against the kernel's <gradient, d>: the gradient's own
    bound, plus the differences' h^2 term."""
    lens, kw = [270, 35], dict(window=40, sinks=2)
    q, k, v, do, cu = make(lens, 4, 2, 64, torch.float16, cuda_dev)
    got, bounds = grads(q, k, v, do, cu, **kw), pa.packed64(q, k, v, lens, True, 0.125, do, **kw)
    h = 1e-4
    for i, name in enumerate(("dQ", "dK", "dV")):
        d = torch.randn_like((q, k, v)[i].double())
        at = [q.double(), k.double(), v.double()]
        ends = []
        for s in (h, -h):
            x = list(at)
            x[i] = at[i] + s * d
            ends.append((pa.packed64(x[0], x[1], x[2], lens, True, 0.125, **kw)["O"][0] * do.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        allowed = (bounds[name][1] * d.abs()).sum() + 1e-4 * do.double().norm()
        assert abs(slope - (got[name].double() * d).sum()) <= allowed


def test_another_stream_and_captured_steps(no_device_error, cuda_dev):
    q, k, v, do, cu = make([430, 60], 4, 2, 128, torch.bfloat16, cuda_dev)
    kw = dict(window=70, sinks=4)
    want = grads(q, k, v, do, cu, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grads(q, k, v, do, cu, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in got)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = bsk.attention_varlen(*leaves, cu, **kw)
        out = (o.detach(), *torch.autograd.grad(o, leaves, do))
        del o
    with torch.no_grad():
        for t, x in zip(leaves, (q, k, v)):
            t.copy_(x.flip(0))
    graph.replay()
    want = grads(*(t.flip(0) for t in (q, k, v)), do, cu, **kw)
    assert all(torch.equal(a, b) for a, b in zip(out, want.values()))


def test_refusals(cuda_dev):
    q, k, v, do, cu = make([30], 4, 2, 64, torch.bfloat16, cuda_dev)
    for kw in (dict(window=0), dict(window=-3), dict(window=5, sinks=-1), dict(sinks=2), dict(window=5, causal=False)):
        with pytest.raises(ValueError):
            bsk.attention_varlen(q, k, v, cu, **kw)
