"""Windowed packed attention whose key blocks with sinks are split along their query tiles: gradients against the 64-bit
definition over group sizes, head dims, types, several sequences, sinks that end inside a block and last blocks that are not full."""
import pytest
import torch

from periodicdent42_b200 import _capi
from test_gpu_attention_varlen import grads, make
from test_gpu_attention_window import check

pytestmark = pytest.mark.gpu

SHAPES = [  # lengths, heads, kv heads, window, sinks
    ([2000], 2, 2, 16, 1), ([2000], 4, 1, 64, 130), ([4000], 8, 1, 33, 1), ([1900, 37, 0, 1100, 700], 4, 4, 31, 130),
    ([1500, 2100], 8, 2, 64, 5), ([129, 2500, 128], 8, 1, 16, 128), ([3333], 1, 1, 50, 300), ([1000, 1000, 1000, 7], 12, 4, 40, 1),
    ([2049], 5, 1, 20, 257), ([700, 1800], 16, 1, 64, 3), ([50] * 20 + [1500], 2, 1, 17, 60),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G,window,sinks", SHAPES)
def test_against_definition(no_device_error, cuda_dev, lens, H, G, D, dtype, window, sinks):
    T, B = sum(lens), len(lens)
    lib = _capi.lib()
    assert lib.bsk_attention_varlen_window_workspace_bytes(T, B, H, G, D, window, sinks, 1) > \
        lib.bsk_attention_varlen_workspace_bytes(T, B, H, G, D, 1) + 65536, "not a shape that is split"
    q, k, v, do, cu = make(lens, H, G, D, dtype, cuda_dev, seed=H + D + window)
    got = grads(q, k, v, do, cu, window=window, sinks=sinks)
    check(got, q, k, v, do, lens, window, sinks)
    again = grads(q, k, v, do, cu, window=window, sinks=sinks)
    assert all(torch.equal(again[n], got[n]) for n in got)  # deterministic


def test_rows_behind_the_last_sequence_and_bad_offsets(cuda_dev):
    """Rows behind the last sequence are zero and reach nothing; offsets past the rows are clamped and reported."""
    q, k, v, do, cu = make([1900, 300], 4, 2, 64, torch.bfloat16, cuda_dev)
    kw = dict(window=24, sinks=9)
    want = grads(q[:1900], k[:1900], v[:1900], do[:1900], cu[:2], **kw)
    for t in (q, k, v, do):
        t[1900:] = float("nan")
    got = grads(q, k, v, do, cu[:2], **kw)
    for n in got:
        assert torch.equal(got[n][:1900], want[n]) and (got[n][1900:] == 0).all(), n
    assert _capi.device_error() == 0
    far = cu.clone()
    far[2] = 10 ** 6
    for t in (q, k, v, do):
        t[1900:] = 1.0
    assert all(torch.isfinite(t).all() for t in grads(q, k, v, do, far, **kw).values())
    assert _capi.device_error() != 0


def test_captured_steps_follow_the_lengths(no_device_error, cuda_dev):
    """A replayed step splits by the lengths as they are then."""
    from periodicdent42_b200 import attention_varlen

    q, k, v, do, cu = make([2200, 100], 4, 1, 64, torch.float16, cuda_dev)
    kw = dict(window=20, sinks=140)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up
        torch.autograd.grad(attention_varlen(*leaves, cu, **kw), leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        o = attention_varlen(*leaves, cu, **kw)
        out = (o.detach(), *torch.autograd.grad(o, leaves, do))
        del o
    for lens in ([2200, 100], [150, 2150], [1, 1]):
        cu.copy_(torch.tensor([0, lens[0], sum(lens)]))
        graph.replay()
        got = dict(zip(("O", "dQ", "dK", "dV"), out))
        n = sum(lens)
        check({m: t[:n] for m, t in got.items()}, *(t.detach()[:n] for t in (q, k, v, do)), lens, 20, 140)
        assert all((t[n:] == 0).all() for t in out)
