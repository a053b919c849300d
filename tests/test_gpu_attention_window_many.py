"""Single tokens and drafts of many sequences over a paged cache with a window, where the warps of a block follow the rounds that
the tiles take: 2, 3 and 4 of them, both cache types, against the 64-bit definition."""
import pytest
import torch

import periodicdent42_b200 as bsk
from test_gpu_attention_paged import make
from test_gpu_attention_window_paged import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("B,H,G,D,page,window,sinks,dtype", [
    (24, 8, 8, 128, 16, 100, 0, torch.bfloat16), (40, 16, 8, 64, 64, 300, 4, torch.float16), (60, 8, 8, 128, 32, 64, 40, torch.bfloat16),
    (64, 16, 8, 128, 16, 513, 1, torch.float16), (75, 8, 8, 64, 8, 1, 3, torch.bfloat16), (100, 16, 8, 128, 128, 257, 130, torch.bfloat16),
    (100, 8, 8, 64, 16, 40, 0, torch.float16), (300, 4, 1, 128, 16, 90, 5, torch.bfloat16),
])
@pytest.mark.parametrize("drafts", [False, True])
def test_against_definition(no_device_error, cuda_dev, B, H, G, D, page, window, sinks, dtype, e4m3, drafts):
    assert B * G > torch.cuda.get_device_properties(cuda_dev).multi_processor_count
    new = [1 + (i % 3 == 1) - (i % 7 == 3) if drafts else 1 for i in range(B)]  # (none, one or two new tokens)
    kv = [max(n, (37 * i * i + 11 * i) % 901) for i, n in enumerate(new)]
    q, c, table, lens, cu = make(new, kv, H, G, D, page, dtype, cuda_dev, e4m3, seed=B)
    kw = dict(window=window, sinks=sinks, **c)
    out = bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw)
    check(out, q, c, table, kv, new, window, sinks)
    assert torch.equal(out, bsk.attention_paged(q, block_table=table, kv_lens=lens, cu_seqlens=cu, **kw))
