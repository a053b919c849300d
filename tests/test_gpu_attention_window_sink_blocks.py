"""Non-finite rows that share a 128-key block with a sink and are none themselves: rows that have left them behind, however far, keep
their results, and so do the gradients of queries; the gradients of keys and values are reached within that block alone."""
import pytest
import torch

import periodicdent42_b200 as bsk
from test_gpu_attention_paged import make as make_paged
from test_gpu_attention_varlen import grads, make

pytestmark = pytest.mark.gpu

# tokens, heads, kv heads, window, sinks, bad rows (behind the sinks, in their last block)
CASES = [(900, 4, 2, 100, 3, (50, 127)), (2000, 4, 1, 60, 130, (130, 255)), (700, 3, 3, 20, 1, (1, 60)), (1500, 8, 1, 300, 127, (127,)),
         (1100, 5, 1, 130, 200, (200, 201, 255))]


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("T,H,G,window,sinks,rows", CASES)
def test_packed(no_device_error, cuda_dev, T, H, G, window, sinks, rows, D, dtype, bad):
    lens = [70, T, 300]
    q, k, v, do, cu = make(lens, H, G, D, dtype, cuda_dev, seed=T)
    kw = dict(window=window, sinks=sinks)
    want = grads(q, k, v, do, cu, **kw)
    keep = torch.ones(sum(lens), dtype=torch.bool, device=cuda_dev)
    keep[70 + max(min(rows) - 255, 0):70 + max(rows) + window + 255] = False  # rows near those that see them
    assert keep[70:70 + T].any()
    at = [70 + r for r in rows]
    for name, reached in (("v", ("O", "dQ")), ("k", ("O", "dQ"))):
        x = dict(q=q, k=k, v=v)
        x[name] = x[name].clone()
        x[name][at] = bad
        got = grads(x["q"], x["k"], x["v"], do, cu, **kw)
        for n in reached:
            assert torch.equal(got[n][keep], want[n][keep]), (name, n)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("T,H,G,window,sinks", [case[:5] for case in CASES])
def test_far_queries_reach_the_sinks_blocks_keys_alone(no_device_error, cuda_dev, T, H, G, window, sinks, D, dtype):
    q, k, v, do, cu = make([T], H, G, D, dtype, cuda_dev, seed=T)
    kw = dict(window=window, sinks=sinks)
    want = grads(q, k, v, do, cu, **kw)
    row = T - 30
    keep = torch.ones(T, dtype=torch.bool, device=cuda_dev)
    keep[:-(-sinks // 128) * 128] = False
    keep[max(row - window - 255, 0):row + 256] = False
    for name in ("q", "do"):
        x = dict(q=q.clone(), do=do.clone())
        x[name][row] = float("nan")
        got = grads(x["q"], k, v, x["do"], cu, **kw)
        for n in ("dK", "dV"):
            assert torch.equal(got[n][keep], want[n][keep]), (name, n)
        assert torch.isnan(got["dK"][:sinks]).any()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,kv,window,sinks,page,row", [
    ([200], [900], 100, 3, 16, 9), ([200], [900], 100, 3, 128, 90), ([90, 300], [700, 2000], 64, 130, 64, 180), ([70], [9000], 3000, 5, 32, 31),
    ([1], [900], 100, 3, 64, 50), ([3, 1], [900, 400], 30, 1, 256, 100), ([400], [400], 10, 20, 16, 25),
])
def test_paged(no_device_error, cuda_dev, new, kv, window, sinks, page, row, e4m3):
    q, c, table, lens, cu = make_paged(new, kv, 8, 2, 128, page, torch.bfloat16, cuda_dev, e4m3, seed=row)
    at = dict(block_table=table, kv_lens=lens, cu_seqlens=cu, window=window, sinks=sinks)
    want = bsk.attention_paged(q, **at, **c)
    for i in range(len(kv)):
        c["v_scale" if e4m3 else "v_cache"][table[i, row // page], row % page] = float("nan")
    got = bsk.attention_paged(q, **at, **c)
    a = 0
    for n, L in zip(new, kv):
        first = max(row + window + 255 - (L - n), 0)  # the first new token well behind those that see it
        assert torch.equal(got[a + first:a + n], want[a + first:a + n])
        a += n
    assert torch.isfinite(want).all()
