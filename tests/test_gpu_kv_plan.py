"""Slots, positions, block tables and lengths of a serving step against the definition, request by request: page ends, empty
requests, more requests and rows than a CTA takes, padding, calls repeated and captured, every reported error, refusals; and the
whole serving step with the operators that use it."""
import random

import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def make(kv, new, page, dev, spare=3, wide=1, seed=0, stale=5):
    """(tensors of a call, lists for the definition): pages in random order, the stack followed by stale entries."""
    rng = random.Random(seed)
    have, need = [-(-k // page) for k in kv], [-(-(k + n) // page) for k, n in zip(kv, new)]
    pages = list(range(sum(need) + spare))
    rng.shuffle(pages)
    width = max([1] + need) + wide
    table, a = [], 0
    for h in have:
        table.append(pages[a:a + h] + [-1] * (width - h))
        a += h
    stack = pages[a:]
    i32 = dict(dtype=torch.int32, device=dev)
    t = dict(kv_lens=torch.tensor(kv, **i32), new_lens=torch.tensor(new, **i32),
             block_table=torch.tensor(table, **i32).view(len(kv), width), free_pages=torch.tensor(stack + [7] * stale, **i32),
             free_count=torch.tensor([len(stack)], **i32))
    return t, table, stack


def check(out, t, kv, new, table, stack, page, tokens):
    want = pa.plan_steps(kv, new, table, stack, page, tokens)
    slots, positions, cu, lens, left = out
    assert slots.dtype == torch.int64 and all(x.dtype == torch.int32 for x in out[1:])
    assert slots.tolist() == want[0] and positions.tolist() == want[1] and cu.tolist() == want[2] and lens.tolist() == want[3]
    assert left.tolist() == [len(want[4])] and t["block_table"].tolist() == want[5]


STEPS = [  # cached, new, page, padding rows
    ([0], [1], 16, 0), ([15], [1], 16, 0), ([16], [1], 16, 3), ([5, 0, 16, 31], [1, 40, 0, 2], 16, 7), ([0, 0], [0, 0], 8, 4),
    ([0, 0], [0, 0], 8, 0), ([1000], [3000], 64, 100), ([7] * 64, [1] * 64, 8, 0), ([3, 100], [1, 1], 1, 2), ([10, 20], [90, 5], 100, 0),
    ([0] * 700, [3] * 700, 16, 13), ([i % 41 for i in range(1600)], [(i * 7) % 5 for i in range(1600)], 8, 1),
    ([0] * 513, [0] * 512 + [9], 4, 0), ([0], [5000], 1024, 0), ([129] * 3 + [0] * 1200, [1030, 0, 2] + [0, 1] * 600, 128, 600),
]


@pytest.mark.parametrize("kv,new,page,padding", STEPS)
def test_against_definition(no_device_error, cuda_dev, kv, new, page, padding):
    tokens = sum(new) + padding
    t, table, stack = make(kv, new, page, cuda_dev, seed=page)
    out = bsk.kv_cache_plan(**t, page_size=page, tokens=tokens)
    check(out, t, kv, new, table, stack, page, tokens)
    again = bsk.kv_cache_plan(**t, page_size=page, tokens=tokens)  # nothing that a call reads is changed by it
    check(again, t, kv, new, table, stack, page, tokens)
    t["kv_lens"], t["new_lens"] = t["kv_lens"].long(), t["new_lens"].long()
    check(bsk.kv_cache_plan(**t, page_size=page, tokens=tokens), t, kv, new, table, stack, page, tokens)


def test_every_free_page_taken_and_strided_table(no_device_error, cuda_dev):
    kv, new = [3, 0, 40], [50, 16, 9]
    t, table, stack = make(kv, new, 16, cuda_dev, spare=0)
    big = torch.full((3, t["block_table"].shape[1] + 9), -5, dtype=torch.int32, device=cuda_dev)
    view = big[:, 4:4 + t["block_table"].shape[1]]
    view.copy_(t["block_table"])
    t["block_table"] = view
    out = bsk.kv_cache_plan(**t, page_size=16, tokens=75)
    check(out, t, kv, new, table, stack, 16, 75)
    assert out[4].item() == 0 and (big[:, :4] == -5).all() and (big[:, -5:] == -5).all()


def test_steps_in_a_captured_graph(no_device_error, cuda_dev):
    """A replayed step follows the lengths and the stack as they are then, its own outputs among them."""
    page, kv, new = 8, [3, 0, 21], [2, 9, 1]
    t, table, stack = make(kv, [200] * 3, page, cuda_dev)
    t["new_lens"].copy_(torch.tensor(new, dtype=torch.int32))
    bsk.kv_cache_plan(**t, page_size=page, tokens=20)  # (the table's entries are written again below)
    t["block_table"].copy_(torch.tensor(table, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bsk.kv_cache_plan(**t, page_size=page, tokens=20)
        t["kv_lens"].copy_(out[3])
        t["free_count"].copy_(out[4])
    for new in ([2, 9, 1], [1, 1, 1], [0, 8, 12], [7, 7, 6]):
        t["new_lens"].copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        check(out, t, kv, new, table, stack, page, 20)
        _, _, _, kv, stack, table = pa.plan_steps(kv, new, table, stack, page, 20)


def test_results_are_tensors_of_their_own(no_device_error, cuda_dev):
    """In inference mode and out of it: results may be changed in place, and a change of one leaves the others."""
    kv, new = [3, 0, 21], [2, 9, 1]
    for mode in (torch.inference_mode, torch.enable_grad):
        with mode():
            t, table, stack = make(kv, new, 8, cuda_dev)
            out = bsk.kv_cache_plan(**t, page_size=8, tokens=15)
            keep = [x.tolist() for x in out]
            for i, x in enumerate(out):
                assert x.is_contiguous() and not x.requires_grad
                x += 1
                assert x.tolist() == [y + 1 for y in keep[i]]
                x -= 1
            assert [x.tolist() for x in out] == keep
            check(out, t, kv, new, table, stack, 8, 15)


def test_two_streams_at_once(no_device_error, cuda_dev):
    """Calls of all the serving operators side by side on two streams give what they give one after the other."""
    torch.manual_seed(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    f, _ = bsk.rotary_frequencies(64, device=cuda_dev)
    w = torch.rand(64, device=cuda_dev).add(0.5).bfloat16()

    def step(seed, lens):
        t, _, _ = make(lens, [n % 7 + 1 for n in lens], 8, cuda_dev, seed=seed)
        rows = sum(n % 7 + 1 for n in lens)
        slots, pos, cu, kv, _ = bsk.kv_cache_plan(**t, page_size=8, tokens=rows)
        g = torch.Generator(device=cuda_dev).manual_seed(seed)
        q, k, v = (torch.randn(rows, h, 64, generator=g, device=cuda_dev).bfloat16() for h in (4, 2, 2))
        pages = int(t["free_pages"].max()) + int(t["block_table"].max()) + 2
        cache = [torch.randn(pages, 8, 2, 64, generator=g, device=cuda_dev).bfloat16() for _ in range(2)]
        q, k = bsk.qk_norm_rotary(q, k, w, w, pos, f)
        bsk.kv_cache_append(k, v, *cache, slots)
        return bsk.attention_paged(q, *cache, t["block_table"], kv, cu, window=20, sinks=2)

    jobs = [(1, [5, 90, 400]), (2, [33] * 40)]
    want = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(step(*j))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


def reported():
    with pytest.raises(RuntimeError):
        bsk.synchronize_and_check()


def test_what_goes_wrong_is_reported(cuda_dev):
    assert _capi.device_error() == 0
    # too few free pages: the requests in front get theirs
    t, table, stack = make([0, 0, 5], [20, 20, 1], 16, cuda_dev, spare=0)
    t["free_count"] -= 2
    slots, pos, cu, lens, left = bsk.kv_cache_plan(**t, page_size=16, tokens=41)
    reported()
    short = stack[:-2]
    want = [short[-1] * 16 + i for i in range(16)] + [short[-2] * 16 + i for i in range(4)] if len(short) > 1 else None
    assert want and slots[:20].tolist() == want and (slots[20:40] == -1).all() and slots[40] == table[2][0] * 16 + 5
    assert t["block_table"][1, :2].tolist() == [-1, -1] and left.item() == 0 and cu.tolist() == [0, 20, 40, 41] and lens.tolist() == [20, 20, 6]
    assert pos.tolist() == [*range(20), *range(20), 5]
    # lengths: negative, past the table, past the rows
    t, table, stack = make([4, 4], [4, 4], 4, cuda_dev, wide=0)
    for kv, new in (([-3, 4], [4, 4]), ([4, 4], [-1, 4]), ([4, 4], [4, 9]), ([2 ** 31 - 1, 4], [2 ** 31 - 1, 4]), ([4, 4], [2 ** 31 - 1, 2 ** 31 - 1])):
        t["kv_lens"].copy_(torch.tensor(kv, dtype=torch.int32))
        t["new_lens"].copy_(torch.tensor(new, dtype=torch.int32))
        slots, pos, cu, lens, left = bsk.kv_cache_plan(**t, page_size=4, tokens=13)
        reported()
        cap = (sum(max(n, 0) for n in new) >= 13)
        assert cu[0] == 0 and (cu[1:] >= cu[:-1]).all() and cu[-1] <= 13 and (lens >= 0).all() and (lens <= 8).all() and (cap or cu[-1] < 13)
        assert (slots >= -1).all() and (slots < 4 * 7).all() and 0 <= left.item() <= len(stack)
    # the stack's size
    t, table, stack = make([0], [3], 4, cuda_dev, stale=0)
    for n in (-1, 10 ** 6):
        t["free_count"].fill_(n)
        slots = bsk.kv_cache_plan(**t, page_size=4, tokens=3)[0]
        reported()
        assert slots.tolist() == ([-1] * 3 if n < 0 else [stack[-1] * 4 + i for i in range(3)])
    # the request's own page was given back
    t, table, stack = make([5], [2], 4, cuda_dev)
    t["block_table"][0, 1] = -1
    assert bsk.kv_cache_plan(**t, page_size=4, tokens=2)[0].tolist() == [-1, -1]
    reported()
    bsk.synchronize_and_check()


def test_refusals(cuda_dev):
    t, _, _ = make([4, 4], [1, 1], 4, cuda_dev)
    good = dict(**t, page_size=4, tokens=2)
    for change in (dict(kv_lens=t["kv_lens"][:1]), dict(new_lens=t["new_lens"].float()), dict(new_lens=t["new_lens"].cpu()),
                   dict(block_table=t["block_table"].long()), dict(block_table=t["block_table"][0]), dict(block_table=t["block_table"].cpu()),
                   dict(block_table=t["block_table"][:1].expand(2, -1)), dict(block_table=t["block_table"].t().contiguous().t()),
                   dict(free_pages=t["free_pages"].long()), dict(free_count=t["free_pages"][:2]), dict(free_count=t["free_count"][0]),
                   dict(page_size=0), dict(page_size=-4), dict(tokens=-1)):
        with pytest.raises(ValueError):
            bsk.kv_cache_plan(**{**good, **change})
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    none = bsk.kv_cache_plan(torch.empty(0, **i32), torch.empty(0, **i32), torch.empty(0, 5, **i32), t["free_pages"], t["free_count"], 4, 3)
    assert none[0].tolist() == [-1] * 3 and none[1].tolist() == [0] * 3 and none[2].tolist() == [0] and none[4].tolist() == t["free_count"].tolist()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,H,G,D,page,window,sinks", [(torch.bfloat16, 8, 2, 128, 16, 60, 4), (torch.float16, 6, 6, 64, 8, 33, 0)])
def test_serving_steps_together(no_device_error, cuda_dev, e4m3, dtype, H, G, D, page, window, sinks):
    """Plan, norm with rotation, cache and windowed attention, chunk by chunk to single tokens, in padded rows -- against the
    definition of attention over the cached rows."""
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    B, pages, width = 3, 80, 40
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    table, kv = torch.full((B, width), -1, **i32), torch.zeros(B, **i32)
    free, count = torch.randperm(pages, generator=g, device=cuda_dev).int(), torch.tensor([pages], **i32)
    f, _ = bsk.rotary_frequencies(D, device=cuda_dev)
    qw, kw = (torch.rand(D, generator=g, device=cuda_dev).add(0.5).to(dtype) for _ in range(2))
    kind = torch.float8_e4m3fn if e4m3 else dtype
    shape = (pages, page, G, D)
    c = dict(k_cache=torch.zeros(shape, device=cuda_dev).to(kind), v_cache=torch.zeros(shape, device=cuda_dev).to(kind))
    if e4m3:
        c.update(k_scale=torch.zeros(shape[:3], device=cuda_dev), v_scale=torch.zeros(shape[:3], device=cuda_dev))
    done = [0] * B
    for step in ([100, 7, 128], [49, 33, 0], [1, 1, 1], [1, 1, 1]):
        rows = sum(step) + 9  # padded
        q, k, v = (torch.randn(rows, n, D, generator=g, device=cuda_dev).to(dtype) for n in (H, G, G))
        slots, pos, cu, kv, count = bsk.kv_cache_plan(kv, torch.tensor(step, **i32), table, free, count, page, rows)
        qr, kr = bsk.qk_norm_rotary(q, k, qw, kw, pos, f)
        bsk.kv_cache_append(kr, v, slots=slots, **c)
        o = bsk.attention_paged(qr, block_table=table, kv_lens=kv, cu_seqlens=cu, window=window, sinks=sinks, **c)
        done = [a + b for a, b in zip(done, step)]
        assert kv.tolist() == done and (o[sum(step):] == 0).all()
        T = sum(step)
        want = pa.norm_rotary64(q, qw, pos, f, False, 1.0, 1e-6)["y"]
        assert pa.worst(qr, *want) <= 1.0
        if not e4m3:
            kept = bsk.kv_cache_gather(slots=slots[:T], dtype=dtype, **c)
            assert torch.equal(kept[0], kr[:T]) and torch.equal(kept[1], v[:T])
        want = pa.paged64(qr[:T], c["k_cache"], c["v_cache"], table, done, step, D ** -0.5, c.get("k_scale"), c.get("v_scale"),
                          window, sinks)
        assert pa.worst(o[:T], *want) <= 1.0


def test_training_step_through_norm_and_windowed_attention(no_device_error, cuda_dev):
    """Gradients through both operators together against torch's autograd of the 64-bit chain."""
    lens, H, G, D, window, sinks = [290, 47], 4, 2, 64, 50, 2
    T = sum(lens)
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    x = [torch.randn(T, n, D, generator=g, device=cuda_dev).half().requires_grad_(True) for n in (H, G, G)]
    w = [torch.rand(D, generator=g, device=cuda_dev).add(0.5).requires_grad_(True) for _ in range(2)]
    do = torch.randn(T, H, D, generator=g, device=cuda_dev).half()
    pos = torch.cat([torch.arange(n, device=cuda_dev) for n in lens])
    f, _ = bsk.rotary_frequencies(D, device=cuda_dev)
    cu = torch.tensor([0, *lens], device=cuda_dev).cumsum(0).int()
    qr, kr = bsk.qk_norm_rotary(x[0], x[1], *w, pos, f)
    got = torch.autograd.grad(bsk.attention_varlen(qr, kr, x[2], cu, window=window, sinks=sinks), x + w, do)
    y = [t.detach().double().requires_grad_(True) for t in x + w]

    def chain(t, weight):
        z = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight
        angle = pos.double()[:, None] * f.double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = z[..., : D // 2], z[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    q64, k64, parts, a = chain(y[0], y[3]), chain(y[1], y[4]), [], 0
    for n in lens:
        r = slice(a, a + n)
        s = torch.einsum("qhd,khd->hqk", q64[r], k64[r].repeat_interleave(H // G, 1)) * D ** -0.5
        s = s.masked_fill(~pa.visible(torch.arange(n, device=cuda_dev), n, window, sinks), float("-inf"))
        parts.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), y[2][r].repeat_interleave(H // G, 1)))
        a += n
    want = torch.autograd.grad(torch.cat(parts), y, do.double())
    for a, b in zip(got, want):  # three fp16 roundings in a row (2^-11 each) on sums of many terms: 4 * 2^-11 normwise
        assert (a.double() - b).norm() <= 4 * 2.0 ** -11 * b.norm()
