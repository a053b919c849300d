"""Attention over e4m3 caches where the values' scales differ: between sequences and heads, between keys, and rows of
zeros -- against the 64-bit definition, elementwise within the roundings' bound."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu


def make(new, kv, H, G, D, page, dtype, dev, seed, value_size):
    """Inputs of one call over an e4m3 cache, pages in random order; value_size [sequences, longest, kv heads] multiplies
    the value rows. Scales behind a sequence's end are NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need), generator=g, device=dev)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=dev)
    k, v = (torch.randn(sum(need), page, G, D, generator=g, device=dev) for _ in range(2))
    first = 0
    held = torch.zeros(sum(need), page, dtype=torch.bool, device=dev)
    for i, (n, p) in enumerate(zip(kv, need)):
        at = order[first:first + p]
        table[i, :p] = at
        size = torch.ones(p * page, G, device=dev)
        size[:n] = value_size[i, :n]
        v[at] *= size.view(p, page, G, 1)
        held[at] = (torch.arange(p * page, device=dev) < n).view(p, page)
        first += p
    c = {}
    for n, x in (("k", k), ("v", v)):
        c[n + "_cache"], c[n + "_scale"] = pa.quantise_rows(x)
        c[n + "_scale"][~held] = float("nan")
    q = torch.randn(sum(new), H, D, generator=g, device=dev).to(dtype)
    at = dict(block_table=table, kv_lens=torch.tensor(kv, dtype=torch.int32, device=dev),
              cu_seqlens=torch.tensor([0] + new, device=dev).cumsum(0).int())
    return q, c, at


def worst(out, q, c, at, kv, new):
    want = pa.paged64(q, c["k_cache"], c["v_cache"], at["block_table"], kv, new, q.shape[2] ** -0.5, c["k_scale"], c["v_scale"])
    return pa.worst(out, *want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_sequences(no_device_error, cuda_dev, D, dtype):
    """More entries than CTAs several times over, each of a single key block, with values of another size for every
    sequence and head: each entry's results carry its own scale."""
    new = [20 + i % 60 for i in range(100)]
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    size = torch.exp2(torch.randint(-8, 9, (100, 1, 8), generator=g, device=cuda_dev).float()).expand(-1, 80, -1)
    q, c, at = make(new, new, 16, 8, D, 16, dtype, cuda_dev, D, size)
    out = bsk.attention_paged(q, **at, **c)
    assert worst(out, q, c, at, new, new) <= 1.0
    for _ in range(3):
        assert torch.equal(out, bsk.attention_paged(q, **at, **c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_that_grow_along_the_sequence(no_device_error, cuda_dev, dtype):
    """The scale reference moves from block to block (and the outputs so far with it), up and down."""
    new, kv = [700, 60, 90], [900, 700, 90]
    size = torch.exp2(torch.arange(900, device=cuda_dev) // 128 * 2.0 - 6)[None, :, None].repeat(3, 1, 2)
    size[1] = size[1].flip(0)
    q, c, at = make(new, kv, 4, 2, 128, 32, dtype, cuda_dev, 1, size)
    out = bsk.attention_paged(q, **at, **c)
    assert worst(out, q, c, at, kv, new) <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_zeros_among_the_values(no_device_error, cuda_dev, dtype):
    """Value rows of zeros (scale 0) with scores far below zero: all of them zero, and one of three."""
    zero = torch.zeros(1, 300, 2, device=cuda_dev)
    some = (torch.arange(300, device=cuda_dev) % 3 > 0)[None, :, None].float().expand(-1, -1, 2)
    for new, size in ((1, zero), (200, zero), (200, some), (1, some)):  # either kernel
        q, c, at = make([new], [300], 4, 2, 128, 16, dtype, cuda_dev, 2, size)
        q.abs_().add_(2.0).mul_(8.0)
        c["k_cache"].view(torch.uint8).bitwise_or_(0x80)  # every key opposite to every query
        out = bsk.attention_paged(q, **at, **c)
        assert worst(out, q, c, at, [300], [new]) <= 1.0
        if size is zero:
            assert (out == 0).all()
    c["k_scale"][at["block_table"][0, 0], 0] = float("nan")  # 0 x NaN is NaN, as by the definition
    c["v_scale"].zero_()
    assert torch.isnan(bsk.attention_paged(q, **at, **c)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,first", [(100, 100, 20), (70, 300, 260), (90, 5000, 4950), (130, 130, 128)])
def test_values_that_a_row_does_not_see_leave_its_precision(no_device_error, cuda_dev, dtype, new, kv, first):
    """Values from position `first` on are 2^34 times the ones before, whose rows keep their own precision."""
    if dtype == torch.float16:  # (results within the type's normal range)
        big, small = 2.0 ** 10, 2.0 ** -8
    else:
        big, small = 2.0 ** 20, 2.0 ** -14
    size = torch.where(torch.arange(kv, device=cuda_dev) < first, small, big)[None, :, None].expand(-1, -1, 2)
    q, c, at = make([new], [kv], 8, 2, 128, 16, dtype, cuda_dev, 3, size)
    out = bsk.attention_paged(q, **at, **c)
    assert worst(out, q, c, at, [kv], [new]) <= 1.0
    dead = first - (kv - new)  # rows before it see small values only
    assert (out[:dead].abs() < small * 8).all() and (out[dead:].abs().amax((1, 2)) > small * 8).all()


def test_an_infinite_value_scale_leaves_other_rows(no_device_error, cuda_dev):
    """Rows of tiles that end before the infinite value are untouched; rows that see it are not finite."""
    size = torch.ones(1, 400, 2, device=cuda_dev)
    q, c, at = make([400], [400], 4, 2, 64, 16, torch.bfloat16, cuda_dev, 4, size)
    want = bsk.attention_paged(q, **at, **c)
    for bad in (float("inf"), float("nan")):
        c["v_scale"][at["block_table"][0, 300 // 16], 300 % 16] = bad
        out = bsk.attention_paged(q, **at, **c)
        assert torch.equal(out[:256], want[:256]) and not torch.isfinite(out[300:]).any()


@pytest.mark.parametrize("new", [1, 200])  # either kernel
def test_queries_with_one_large_element(no_device_error, cuda_dev, new):
    """A bf16 query whose scores come from elements 2^-31 of its largest (which meets zeros)."""
    q, c, at = make([new], [300], 4, 2, 128, 16, torch.bfloat16, cuda_dev, 5, torch.ones(1, 300, 2, device=cuda_dev))
    q.copy_((1 + q.abs().clamp(max=0.99)).mul(2.0 ** -11) * q.sign())
    q[..., 3] = 2.0 ** 20
    c["k_cache"].view(torch.uint8)[..., 3] = 0
    c["k_scale"] *= 4096.0
    assert worst(bsk.attention_paged(q, **at, **c), q, c, at, [300], [new]) <= 1.0
    q[..., 3] = torch.finfo(torch.bfloat16).max  # the largest bf16 value turns into a finite fp16 value
    assert torch.isfinite(bsk.attention_paged(q, **at, **c)).all()


@pytest.mark.parametrize("H,G,D", [(3, 1, 64), (16, 2, 128), (33, 1, 64)])
def test_chunks_that_start_at_every_place_of_a_block(no_device_error, cuda_dev, H, G, D):
    """Tiles that begin on either side of a key block's end, rows without keys in front of it, several entries per CTA."""
    start = [-2, -1, 0, 1, 41, 126, 127, 128, 129, 254, 255, 256, 382, 383, 384, 511, 639]
    new = [1 + (29 * i) % 90 for i in range(3 * len(start))]
    kv = [max(n + start[i % len(start)], 0) for i, n in enumerate(new)]
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    size = torch.exp2(torch.randint(-6, 7, (len(new), 1, G), generator=g, device=cuda_dev).float()).expand(-1, max(kv), -1)
    q, c, at = make(new, kv, H, G, D, 16, torch.bfloat16, cuda_dev, 6, size)
    out = bsk.attention_paged(q, **at, **c)
    assert worst(out, q, c, at, kv, new) <= 1.0
    for _ in range(3):
        assert torch.equal(out, bsk.attention_paged(q, **at, **c))
