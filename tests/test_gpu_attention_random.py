"""Drawn calls of the packed and paged attention against the 64-bit definition: batches, lengths, groups, page sizes, cache types
and value sizes in combinations that nobody listed; every call repeated bit for bit, rows behind the last sequence zero."""
import random

import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu


def _heads(rng):
    kv_heads, group = rng.choice([(1, 1), (3, 2), (2, 3), (8, 4), (3, 5), (1, 7), (2, 8), (3, 16), (1, 33), (1, 128)])
    return kv_heads, group * kv_heads, rng.choice([64, 128]), rng.choice([torch.bfloat16, torch.float16])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seed", range(8))
def test_paged(no_device_error, cuda_dev, seed, e4m3):
    rng, g = random.Random(seed), torch.Generator(device=cuda_dev).manual_seed(seed)
    G, H, D, dtype = _heads(rng)
    page, batch = rng.choice([8, 16, 32, 64, 256, 1024]), rng.choice([1, 2, 7, 40])
    most, longest = rng.choice([1, 3, 40, 200 if batch < 40 else 60]), rng.choice([20, 130, 400, 3000 if batch < 40 else 200])
    new = [rng.choice([0, 1, rng.randint(1, most), most]) for _ in range(batch)]
    new[0] = max(new[0], 1)
    kv = [max(0, n + rng.randint(-2, longest)) for n in new]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device=cuda_dev)
    table = torch.full((batch, max([1] + need) + rng.randint(0, 3)), -1, dtype=torch.int32, device=cuda_dev)
    first = 0
    for i, p in enumerate(need):
        table[i, :p] = order[first:first + p]
        first += p
    k, v = (torch.randn(pages, page, G, D, generator=g, device=cuda_dev) for _ in range(2))
    c = {}
    if e4m3:
        per = rng.choice([(pages, page, G, 1), (pages, 1, 1, 1), (1, 1, G, 1)])  # by row, by page, by head
        v *= torch.exp2(torch.randint(-6 if dtype == torch.float16 else -20, 3, per, generator=g, device=cuda_dev).float())
        if rng.random() < 0.3:
            v *= torch.rand(pages, page, G, 1, generator=g, device=cuda_dev) < 0.5
        for n, x in (("k", k), ("v", v)):
            c[n + "_cache"], c[n + "_scale"] = pa.quantise_rows(x)
    else:
        c = dict(k_cache=k.to(dtype), v_cache=v.to(dtype))
    total, pad = sum(new), rng.choice([0, 5])
    q = (torch.randn(total + pad, H, D, generator=g, device=cuda_dev) * rng.choice([0.3, 1, 3])).to(dtype)
    at = dict(block_table=table, kv_lens=torch.tensor(kv, device=cuda_dev), cu_seqlens=torch.tensor([0] + new, device=cuda_dev).cumsum(0))
    out = bsk.attention_paged(q, **at, **c)
    want = pa.paged64(q[:total], c["k_cache"], c["v_cache"], table, kv, new, D ** -0.5, c.get("k_scale"), c.get("v_scale"))
    assert pa.worst(out[:total], *want) <= 1.0 and (out[total:] == 0).all()
    for _ in range(2):
        assert torch.equal(out, bsk.attention_paged(q, **at, **c))


@pytest.mark.parametrize("seed", range(8))
def test_packed(no_device_error, cuda_dev, seed):
    rng, g = random.Random(seed), torch.Generator(device=cuda_dev).manual_seed(seed)
    G, H, D, dtype = _heads(rng)
    batch = rng.choice([1, 2, 5, 20])
    longest = rng.choice([1, 40, 130, 400 if batch < 20 else 90])
    lens = [rng.choice([0, 1, rng.randint(1, longest), longest]) for _ in range(batch)]
    total, causal = sum(lens), rng.random() < 0.7
    T = total + rng.choice([0, 9])
    q, do = ((torch.randn(T, H, D, generator=g, device=cuda_dev) * s).to(dtype) for s in (rng.choice([0.3, 1, 3]), 1))
    k, v = (torch.randn(T, G, D, generator=g, device=cuda_dev).to(dtype) for _ in range(2))
    cu = torch.tensor([0] + lens, device=cuda_dev).cumsum(0)

    def run():
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = bsk.attention_varlen(*x, cu, causal=causal)
        return (o.detach(), *torch.autograd.grad(o, x, do))

    got = run()
    want = pa.packed64(q[:total], k[:total], v[:total], lens, causal, D ** -0.5, do[:total])
    for x, name in zip(got, ("O", "dQ", "dK", "dV")):
        assert pa.worst(x[:total], *want[name]) <= 1.0 and (x[total:] == 0).all(), name
    assert all(torch.equal(a, b) for a, b in zip(got, run()))
