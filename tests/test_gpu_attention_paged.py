"""Attention of new tokens over a paged cache against its 64-bit definition, elementwise within the roundings' bound:
one to many new tokens, group sizes, page sizes, cache types, empty rows, stale pages, strides, streams, graphs, bad
indices, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def make(new, kv, H, G, D, page, dtype, dev, e4m3=False, seed=0, spare=2, wide=1):
    """Inputs of one call: randomly placed pages, every cache byte behind a sequence's end NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in kv]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=dev)
    width = max([1] + need) + wide
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device=dev)
    x = [torch.randn(pages, page, G, D, generator=g, device=dev) for _ in range(2)]
    held = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    a = 0
    for i, (n, p) in enumerate(zip(kv, need)):
        table[i, :p] = order[a:a + p]
        for j in range(p):
            held[order[a + j], : min(page, n - j * page)] = True
        a += p
    c = {"k_cache": None, "v_cache": None}
    if e4m3:
        for n, y in zip("kv", x):
            c[n + "_cache"], c[n + "_scale"] = pa.quantise_rows(y)
            c[n + "_scale"][~held] = float("nan")
    else:
        for n, y in zip("kv", x):
            c[n + "_cache"] = y.to(dtype)
            c[n + "_cache"][~held] = float("nan")
    q = torch.randn(sum(new), H, D, generator=g, device=dev).to(dtype)
    cu = torch.tensor([0] + new, device=dev).cumsum(0).int()
    return q, c, table, torch.tensor(kv, dtype=torch.int32, device=dev), cu


def check(out, q, c, table, kv, new, scale=None):
    want, bound = pa.paged64(q, c["k_cache"], c["v_cache"], table, kv, new, scale or q.shape[2] ** -0.5, c.get("k_scale"),
                             c.get("v_scale"))
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    assert pa.worst(out, want, bound) <= 1.0


SHAPES = [  # new tokens, cached tokens, heads, kv heads, page
    ([1], [1], 1, 1, 16), ([1], [517], 32, 8, 16), ([1, 1, 1], [5, 700, 64], 8, 8, 64), ([1] * 5, [64, 1, 333, 128, 17], 12, 2, 32),
    ([8] * 3, [1000, 8, 77], 16, 4, 128), ([5, 0, 1, 3], [5, 9, 0, 130], 10, 2, 8), ([130, 7], [400, 7], 6, 2, 64),
    ([300], [1200], 4, 1, 256), ([64, 1, 17], [2000, 1, 17], 5, 5, 16), ([2], [40], 128, 1, 16), ([3, 200], [1, 150], 4, 2, 1024),
    ([1, 40], [4100, 3000], 24, 8, 32),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,kv,H,G,page", SHAPES)
def test_against_definition(no_device_error, cuda_dev, new, kv, H, G, page, D, dtype, e4m3):
    q, c, table, lens, cu = make(new, kv, H, G, D, page, dtype, cuda_dev, e4m3, seed=len(new) + D)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
    check(out, q, c, table, kv, new)
    assert torch.equal(out, bsk.attention_paged(q, block_table=table.long(), kv_lens=lens.long(), cu_seqlens=cu.long(), **c))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,kv,H,G,D,page", [
    ([2500], [2600], 32, 8, 64, 64),           # more tiles than CTAs twice over: nothing is split
    ([70], [9000], 4, 2, 128, 32),             # few tiles, long keys: split many ways
    ([33, 300, 1, 90], [5000, 310, 4096, 90], 8, 1, 64, 16),  # split and whole entries side by side
    ([200, 40], [0, 3000], 4, 4, 128, 16),     # entries without keys beside split ones
])
def test_split_and_whole_entries(no_device_error, cuda_dev, new, kv, H, G, D, page, e4m3):
    q, c, table, lens, cu = make(new, kv, H, G, D, page, torch.bfloat16, cuda_dev, e4m3)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
    check(out, q, c, table, kv, new)
    for _ in range(2):  # the list's order may differ between calls, the results do not
        assert torch.equal(out, bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_and_scale(no_device_error, cuda_dev, dtype):
    q, c, table, lens, cu = make([3, 150], [900, 700], 8, 2, 128, 16, dtype, cuda_dev)
    q = q * 8
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, scale=0.2, **c)
    check(out, q, c, table, [900, 700], [3, 150], 0.2)


def test_rows_without_keys_and_padding_rows_are_zero(no_device_error, cuda_dev):
    for new, kv in (([4, 2], [2, 0]), ([300, 200], [100, 0])):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 16, torch.bfloat16, cuda_dev)
        padded = torch.cat([q, torch.full((37, 4, 64), float("nan"), device=cuda_dev, dtype=q.dtype)])
        out = bsk.attention_paged(padded, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        T, dead = sum(new), new[0] - kv[0]
        check(out[:T], q, c, table, kv, new)
        assert (out[:dead] == 0).all() and (out[new[0]:] == 0).all() and (out[dead:new[0]] != 0).any()
    out = bsk.attention_paged(padded, block_table=table[:0], kv_lens=lens[:0], cu_seqlens=cu[:1], **c)
    assert (out == 0).all()  # no sequences at all
    assert bsk.attention_paged(q[:0], block_table=table, kv_lens=lens, cu_seqlens=cu * 0, **c).shape == (0, 4, 64)


def test_strided_queries(no_device_error, cuda_dev):
    for new, kv in (([2, 3], [33, 50]), ([140, 60], [300, 60])):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 32, torch.float16, cuda_dev)
        want = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        qkv = torch.randn(sum(new), 8, 64, device=cuda_dev).half()
        qkv[:, 2:6] = q
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=cuda_dev)[1:].view_as(q).copy_(q)
        for view in (qkv[:, 2:6], q.transpose(0, 1).contiguous().transpose(0, 1), odd):
            assert torch.equal(bsk.attention_paged(view, block_table=table, kv_lens=lens, cu_seqlens=cu, **c), want)
        one = q[:, :1].expand(-1, 4, -1)
        assert torch.equal(bsk.attention_paged(one, block_table=table, kv_lens=lens, cu_seqlens=cu, **c),
                           bsk.attention_paged(one.contiguous(), block_table=table, kv_lens=lens, cu_seqlens=cu, **c))


def test_wide_table_gives_the_same_definition(no_device_error, cuda_dev):
    """A table with room for a far longer context (its unused entries are never read as pages)."""
    for e4m3 in (False, True):
        q, c, table, lens, cu = make([1, 130], [100, 400], 8, 2, 128, 16, torch.bfloat16, cuda_dev, e4m3, wide=3000)
        check(bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c), q, c, table, [100, 400], [1, 130])


def test_another_stream_and_captured_graph(no_device_error, cuda_dev):
    q, c, table, lens, cu = make([1, 3, 200], [700, 90, 333], 8, 2, 128, 16, torch.bfloat16, cuda_dev)
    want = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graphs = []
    for _ in range(2):  # two graphs of one pool, replayed in turn, with inputs that change between replays
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=graphs[0][0].pool() if graphs else None):
            out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        graphs.append((gr, out))
    for step in range(3):
        q.copy_(torch.randn_like(q))
        lens.copy_(torch.tensor([700 - step, 90, 333 - 7 * step], device=cuda_dev))
        want = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        for gr, out in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("new,kv", [([3], [200]), ([150], [400])])  # either kernel
def test_non_finite_keys_reach_the_rows_that_see_them_only(no_device_error, cuda_dev, new, kv):
    for e4m3 in (False, True):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 16, torch.bfloat16, cuda_dev, e4m3)
        want = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
        p = kv[0] - 2  # seen by the last two new tokens
        page, off = int(table[0, p // 16]), p % 16
        # (a row of infinities gives sums of both signs, NaN; an infinite scale would give +inf or, rightly, -inf: weight 0)
        for bad in (float("nan"),) if e4m3 else (float("nan"), float("inf")):
            if e4m3:
                c["k_scale"][page, off, 1] = bad
            else:
                c["k_cache"][page, off, 1] = bad
            got = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)
            assert torch.equal(got[:-2], want[:-2]) and torch.equal(got[-2:, :2], want[-2:, :2])
            assert torch.isnan(got[-2:, 2:]).all()


def test_cache_behind_two_to_the_31_elements(no_device_error, cuda_dev):
    """Slots whose elements lie more than 2^31 behind the cache's start, written, read back and attended to."""
    G, D, page = 8, 128, 64
    pages = (2 ** 31 // (G * D) + 4096) // page
    c = {n: torch.zeros(pages, page, G, D, dtype=torch.bfloat16, device=cuda_dev) for n in ("k_cache", "v_cache")}
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    L = 700
    k, v = (torch.randn(L, G, D, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    order = pages - 1 - torch.randperm(40, generator=g, device=cuda_dev)[: -(-L // page)]
    at = torch.arange(L, device=cuda_dev)
    slots = order[at // page] * page + at % page
    assert int(slots.min()) * G * D > 2 ** 31
    bsk.kv_cache_append(k, v, slots=slots, **c)
    kr, vr = bsk.kv_cache_gather(slots=slots, **c)
    assert torch.equal(kr, k) and torch.equal(vr, v)
    table = order[None].int()
    for n in (2, 100):
        q = torch.randn(n, 16, D, generator=g, device=cuda_dev).bfloat16()
        out = bsk.attention_paged(q, block_table=table, kv_lens=torch.tensor([L], device=cuda_dev),
                                  cu_seqlens=torch.tensor([0, n], device=cuda_dev), **c)
        allowed = torch.arange(L, device=cuda_dev) <= (L - n + torch.arange(n, device=cuda_dev))[:, None]
        for h in (0, 7, 15):
            want, bound = pa.attention64(q[:, h], k[:, h // 2], v[:, h // 2], allowed, D ** -0.5, q.dtype)[:2]
            assert pa.worst(out[:, h], want, bound) <= 1.0


def test_two_streams_at_once(no_device_error, cuda_dev):
    """Calls that run side by side share nothing: each gives what it gives alone."""
    jobs = [make(new, kv, 8, 2, 128, 16, torch.bfloat16, cuda_dev, e4m3, seed=i)
            for i, (new, kv, e4m3) in enumerate([([40], [5000], False), ([40], [5000], True), ([1] * 9, [3000] * 9, True),
                                                 ([300, 20], [900, 2000], False)])]
    alone = [bsk.attention_paged(q, block_table=t, kv_lens=n, cu_seqlens=u, **c) for q, c, t, n, u in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        outs = []
        for s, (q, c, t, n, u) in zip(streams, jobs):
            with torch.cuda.stream(s):
                outs.append(bsk.attention_paged(q, block_table=t, kv_lens=n, cu_seqlens=u, **c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_bad_indices_are_reported_not_followed(cuda_dev):
    assert _capi.device_error() == 0
    for new, kv in (([1, 2], [40, 70]), ([150, 200], [400, 300])):
        q, c, table, lens, cu = make(new, kv, 4, 2, 64, 16, torch.bfloat16, cuda_dev)
        room = table.shape[1] * 16

        def fails(t=table, n=lens, u=cu):
            bsk.attention_paged(q, block_table=t, kv_lens=n, cu_seqlens=u, **c)
            with pytest.raises(RuntimeError, match="out-of-range"):
                bsk.synchronize_and_check()

        for page in (-1, c["k_cache"].shape[0], 2 ** 31 - 1):
            t = table.clone()
            t[1, 1] = page
            fails(t=t)
        fails(n=torch.tensor([kv[0], room + 1], device=cuda_dev, dtype=torch.int32))
        fails(n=torch.tensor([-3, kv[1]], device=cuda_dev, dtype=torch.int32))
        fails(u=torch.tensor([0, new[0], sum(new) + 5], device=cuda_dev, dtype=torch.int32))
        fails(u=torch.tensor([0, new[0], new[0] - 1], device=cuda_dev, dtype=torch.int32))
        fails(u=torch.tensor([1, new[0], sum(new)], device=cuda_dev, dtype=torch.int32))
        # and the next call is right again
        check(bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c), q, c, table, kv, new)
    assert _capi.device_error() == 0


def test_refusals(cuda_dev):
    q, c, table, lens, cu = make([1, 2], [20, 30], 4, 2, 64, 16, torch.bfloat16, cuda_dev)
    _, e, _, _, _ = make([1, 2], [20, 30], 4, 2, 64, 16, torch.bfloat16, cuda_dev, True)
    base = dict(Q=q, block_table=table, kv_lens=lens, cu_seqlens=cu, **c)

    def cut(page):
        return {n: t[:, :page].contiguous() for n, t in c.items()}

    bad = [dict(Q=q[0]), dict(Q=q.float()), dict(Q=q.half()), dict(Q=q.cpu()), dict(Q=q[..., :32]), dict(Q=q[:, :3]), dict(Q=q[:, :0]),
           dict(block_table=table[0]), dict(block_table=table.float()), dict(block_table=table[:1]), dict(kv_lens=lens[:1]),
           dict(kv_lens=lens.cpu()), dict(cu_seqlens=cu[:2]), dict(cu_seqlens=cu.double()), dict(scale=0.0),
           dict(scale=float("nan")), dict(scale=-1.0), cut(4), cut(12), dict(k_scale=e["k_scale"]),
           dict(k_cache=e["k_cache"], v_cache=e["v_cache"]), dict(k_cache=c["k_cache"].transpose(0, 1))]
    for change in bad:
        with pytest.raises(ValueError):
            bsk.attention_paged(**{**base, **change})
