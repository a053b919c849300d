"""Attention of new tokens over a paged cache with a sliding window and sinks, against the 64-bit definition, elementwise
within the roundings' bound: single tokens, drafts, chunks, both cache types, pages that were given back, values' scales of
keys that a row does not see, rows without keys, graphs, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from test_gpu_attention_paged import make

pytestmark = pytest.mark.gpu


def check(out, q, c, table, kv, new, window, sinks, scale=None):
    want = pa.paged64(q, c["k_cache"], c["v_cache"], table, kv, new, scale or q.shape[2] ** -0.5, c.get("k_scale"),
                      c.get("v_scale"), window, sinks)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    w = pa.worst(out, *want)
    assert w <= 1.0, w


SHAPES = [  # new tokens, cached tokens, heads, kv heads, page, window, sinks
    ([1], [1], 1, 1, 16, 1, 0), ([1], [517], 32, 8, 16, 100, 0), ([1, 1, 1], [5, 700, 64], 8, 8, 64, 64, 4),
    ([1] * 5, [64, 1, 333, 128, 17], 12, 2, 32, 1, 0), ([8] * 3, [1000, 8, 77], 16, 4, 128, 333, 70),
    ([5, 0, 1, 3], [5, 9, 0, 130], 10, 2, 8, 3, 2), ([130, 7], [400, 7], 6, 2, 64, 50, 0), ([300], [1200], 4, 1, 256, 128, 128),
    ([64, 1, 17], [2000, 1, 17], 5, 5, 16, 500, 3), ([2], [40], 128, 1, 16, 9, 1), ([3, 200], [1, 150], 4, 2, 1024, 20, 300),
    ([1, 40], [4100, 3000], 24, 8, 32, 1000, 17), ([700, 300], [5000, 300], 8, 2, 16, 33, 1), ([200], [900], 4, 4, 8, 1, 0),
    ([90], [6000], 8, 2, 64, 2000, 200),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,kv,H,G,page,window,sinks", SHAPES)
def test_against_definition(no_device_error, cuda_dev, new, kv, H, G, page, D, dtype, e4m3, window, sinks):
    q, c, table, lens, cu = make(new, kv, H, G, D, page, dtype, cuda_dev, e4m3, seed=len(new) + D)
    kw = dict(window=window, sinks=sinks, **c)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw)
    check(out, q, c, table, kv, new, window, sinks)
    assert torch.equal(out, bsk.attention_paged(q, block_table=table.long(), kv_lens=lens.long(), cu_seqlens=cu.long(), **kw))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,kv,H,G,D,page,window,sinks", [
    ([2500], [2600], 32, 8, 64, 64, 400, 4),
    ([70], [9000], 4, 2, 128, 32, 5000, 130),
    ([33, 300, 1, 90], [5000, 310, 4096, 90], 8, 1, 64, 16, 2000, 0),
    ([200, 40], [0, 3000], 4, 4, 128, 16, 1500, 1),
])
def test_split_and_whole_entries(no_device_error, cuda_dev, new, kv, H, G, D, page, e4m3, window, sinks):
    q, c, table, lens, cu = make(new, kv, H, G, D, page, torch.bfloat16, cuda_dev, e4m3)
    kw = dict(window=window, sinks=sinks, **c)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw)
    check(out, q, c, table, kv, new, window, sinks)
    for _ in range(2):
        assert torch.equal(out, bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,window,sinks,page", [([1, 1], 100, 3, 16), ([6, 1], 64, 0, 8), ([200, 90], 150, 20, 16), ([300, 5], 10, 1, 32)])
def test_pages_that_were_given_back(no_device_error, cuda_dev, new, window, sinks, page, e4m3):
    """Pages that no new token sees hold another request's NaN, and their table entries are no page numbers: no bit changes
    and no error is reported."""
    kv = [900, 700]
    q, c, table, lens, cu = make(new, kv, 8, 2, 64, page, torch.bfloat16, cuda_dev, e4m3)
    at = dict(block_table=table, kv_lens=lens, cu_seqlens=cu, window=window, sinks=sinks)
    want = bsk.attention_paged(q, **at, **c)
    check(want, q, c, table, kv, new, window, sinks)
    freed = 0
    for i, (n, L) in enumerate(zip(new, kv)):
        first = max(L - n - window + 1, 0)  # the first key that the first new token's window holds
        for p in range(-(-sinks // page), first // page):
            page_no = int(table[i, p])
            for t in ("k_cache", "v_cache") if not e4m3 else ("k_scale", "v_scale"):
                c[t][page_no] = float("nan")
            table[i, p] = (-1, 2 ** 30, -2 ** 31)[freed % 3]
            freed += 1
    assert freed > 10
    assert torch.equal(bsk.attention_paged(q, **at, **c), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,window,sinks,big_from,big_to", [
    (100, 100, 30, 0, 0, 20), (100, 400, 60, 5, 250, 310), (200, 300, 17, 0, 100, 140), (90, 5000, 300, 0, 4500, 4700),
    (150, 200, 128, 1, 0, 1), (40, 300, 50, 40, 30, 60), (1, 300, 50, 0, 200, 250), (8, 300, 20, 3, 250, 277),
])
def test_scales_that_a_row_does_not_see_leave_its_precision(no_device_error, cuda_dev, dtype, new, kv, window, sinks, big_from, big_to):
    """Values at positions [big_from, big_to) are 2^34 (fp16 2^18) times the others: rows that have left them behind, or do not
    reach them yet, keep their own precision."""
    q, c, table, lens, cu = make([new], [kv], 8, 2, 128, 16, dtype, cuda_dev, True, seed=new)
    big, small = (2.0 ** 20, 2.0 ** -14) if dtype == torch.bfloat16 else (2.0 ** 10, 2.0 ** -8)
    place = torch.arange(kv, device=cuda_dev)
    size = torch.where((place >= big_from) & (place < big_to), big, small)
    pages = table[0, place // 16].long()
    c["v_scale"][pages, place % 16] *= size[:, None]
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, window=window, sinks=sinks, **c)
    check(out, q, c, table, [kv], [new], window, sinks)


@pytest.mark.parametrize("H,G,D,window,sinks", [(3, 1, 64, 20, 0), (16, 2, 128, 140, 3), (33, 1, 64, 60, 129)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_chunks_that_start_at_every_place_of_a_block(no_device_error, cuda_dev, H, G, D, window, sinks, e4m3):
    start = [-2, -1, 0, 1, 41, 126, 127, 128, 129, 254, 255, 256, 382, 383, 384, 511, 639]
    new = [1 + (29 * i) % 90 for i in range(3 * len(start))]
    kv = [max(n + start[i % len(start)], 0) for i, n in enumerate(new)]
    q, c, table, lens, cu = make(new, kv, H, G, D, 16, torch.bfloat16, cuda_dev, e4m3, seed=6)
    kw = dict(window=window, sinks=sinks, **c)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw)
    check(out, q, c, table, kv, new, window, sinks)
    for _ in range(3):
        assert torch.equal(out, bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw))


def test_a_window_beyond_the_table_is_plain_causal_attention(no_device_error, cuda_dev):
    for new, kv in (([1, 3], [300, 77]), ([150, 40], [300, 77])):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 16, torch.bfloat16, cuda_dev)
        want = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        for window, sinks in ((10 ** 5, 0), (2 ** 40, 2 ** 40), (2 ** 31 - 1, 5)):
            assert torch.equal(bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, window=window, sinks=sinks,
                                                   **c), want)


def test_rows_without_keys_padding_and_empty_calls(no_device_error, cuda_dev):
    for new, kv in (([4, 2], [2, 0]), ([300, 200], [100, 0])):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 16, torch.bfloat16, cuda_dev)
        padded = torch.cat([q, torch.full((37, 4, 64), float("nan"), device=cuda_dev, dtype=q.dtype)])
        out = bsk.attention_paged(padded, block_table=table, kv_lens=lens, cu_seqlens=cu, window=5, sinks=1, **c)
        T, dead = sum(new), new[0] - kv[0]
        check(out[:T], q, c, table, kv, new, 5, 1)
        assert (out[:dead] == 0).all() and (out[new[0]:] == 0).all() and (out[dead:new[0]] != 0).any()
    assert bsk.attention_paged(q[:0], block_table=table, kv_lens=lens, cu_seqlens=cu * 0, window=5, **c).shape == (0, 4, 64)


def test_captured_graph_with_moving_lengths(no_device_error, cuda_dev):
    """A replayed call follows the lengths and the table as they are then."""
    for new, kv in (([1, 1, 1], [700, 90, 333]), ([60, 3, 200], [700, 90, 333])):
        q, c, table, lens, cu = make(new, kv, 8, 2, 128, 16, torch.bfloat16, cuda_dev, wide=4)
        kw = dict(block_table=table, kv_lens=lens, cu_seqlens=cu, window=120, sinks=4, **c)
        bsk.attention_paged(q, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = bsk.attention_paged(q, **kw)
        shorter = [n - 37 if n > 300 else n for n in kv]
        lens.copy_(torch.tensor(shorter, dtype=torch.int32))
        graph.replay()
        check(out, q, c, table, shorter, new, 120, 4)


def test_refusals(cuda_dev):
    q, c, table, lens, cu = make([2], [30], 4, 2, 64, 16, torch.bfloat16, cuda_dev)
    for kw in (dict(window=0), dict(window=-3), dict(window=5, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw, **c)
    bad = table.clone()
    bad[0, 1] = 10 ** 6  # inside the window: reported
    bsk.attention_paged(q, block_table=bad, kv_lens=lens, cu_seqlens=cu, window=10, **c)
    with pytest.raises(RuntimeError):
        bsk.synchronize_and_check()
