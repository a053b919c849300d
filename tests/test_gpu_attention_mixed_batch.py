"""Single tokens and prompt chunks in one call, the ordinary step of a serving loop, against the 64-bit definition: batches
that either kernel takes, lengths far apart, sequences without new tokens or without keys among them."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu

BATCHES = [  # new tokens, cached tokens
    ([1] * 40 + [300], [17 + 23 * i for i in range(40)] + [900]),          # 8.3 tokens a sequence on average
    ([700] + [1] * 150, [1500] + [1 + 5 * i for i in range(150)]),         # 5.6: a long chunk in small tiles (at 4 heads a group)
    ([1, 0, 256, 1, 1, 0, 33, 1], [4000, 50, 256, 1, 129, 0, 1000, 64]),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,H,G,D,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 4, 1, 64, 64)])
@pytest.mark.parametrize("new,kv", BATCHES)
def test_against_definition(no_device_error, cuda_dev, new, kv, dtype, H, G, D, page, e4m3):
    g = torch.Generator(device=cuda_dev).manual_seed(len(new))
    need = [-(-n // page) for n in kv]
    order = torch.randperm(sum(need), generator=g, device=cuda_dev)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=cuda_dev)
    a = 0
    for i, p in enumerate(need):
        table[i, :p] = order[a:a + p]
        a += p
    k, v = (torch.randn(sum(need), page, G, D, generator=g, device=cuda_dev) for _ in range(2))
    c = {}
    for n, x in (("k", k), ("v", v)):
        if e4m3:
            c[n + "_cache"], c[n + "_scale"] = pa.quantise_rows(x)
        else:
            c[n + "_cache"] = x.to(dtype)
    q = torch.randn(sum(new), H, D, generator=g, device=cuda_dev).to(dtype)
    out = bsk.attention_paged(q, block_table=table, kv_lens=torch.tensor(kv, device=cuda_dev),
                              cu_seqlens=torch.tensor([0] + new, device=cuda_dev).cumsum(0), **c)
    want = pa.paged64(q, c["k_cache"], c["v_cache"], table, kv, new, D ** -0.5, c.get("k_scale"), c.get("v_scale"))
    assert pa.worst(out, *want) <= 1.0
