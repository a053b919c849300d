"""A NaN score reaches the row's result also where the tile goes on to blocks of keys that the row does not see."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H", [3, 5])  # tiles of 42 and 25 tokens: some reach over a block's end
def test_packed(no_device_error, cuda_dev, dtype, H):
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q, k, v = (torch.randn(400, n, 64, generator=g, device=cuda_dev).to(dtype) for n in (H, 1, 1))
    cu = torch.tensor([0, 400], device=cuda_dev)
    want = bsk.attention_varlen(q, k, v, cu)
    k[3, 0, 5] = float("nan")
    got = bsk.attention_varlen(q, k, v, cu)
    assert torch.equal(got[:3], want[:3]) and torch.isnan(got[3:]).all()
    k.requires_grad_(True)  # and with the log-sum-exp kept for the gradients
    o = bsk.attention_varlen(q, k, v, cu)
    assert torch.isnan(o[3:]).all()
    assert torch.isnan(torch.autograd.grad(o, k, torch.ones_like(o))[0]).all()


@pytest.mark.parametrize("kind", ["16-bit", "e4m3"])
@pytest.mark.parametrize("new,kv", [(200, 300), (60, 5000)])  # whole entries, split ones
def test_paged(no_device_error, cuda_dev, kind, new, kv):
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    q = torch.randn(new, 4, 128, generator=g, device=cuda_dev).bfloat16()
    pages = -(-kv // 16)
    k, v = (torch.randn(pages, 16, 2, 128, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
    c = dict(k_cache=k, v_cache=v)
    if kind == "e4m3":
        for n, x in (("k", k), ("v", v)):
            c[n + "_cache"], c[n + "_scale"] = pa.quantise_rows(x)
    at = dict(block_table=torch.arange(pages, device=cuda_dev)[None], kv_lens=torch.tensor([kv], device=cuda_dev),
              cu_seqlens=torch.tensor([0, new], device=cuda_dev))
    want = bsk.attention_paged(q, **at, **c)
    if kind == "e4m3":
        c["k_scale"][0, 7, 0] = float("nan")
    else:
        k[0, 7, 0, 5] = float("nan")
    got = bsk.attention_paged(q, **at, **c)
    assert torch.isnan(got[:, :2]).all() and torch.equal(got[:, 2:], want[:, 2:])
