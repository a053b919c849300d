"""Index tensors in 64 bits: values that 32 bits cannot hold are reported like any other out-of-range value, not wrapped."""
import pytest
import torch

import periodicdent42_b200 as bsk
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def _reported(call):
    call()
    with pytest.raises(RuntimeError, match="out-of-range"):
        bsk.synchronize_and_check()


@pytest.mark.parametrize("n,L", [(3, 40), (150, 300)])  # either kernel
@pytest.mark.parametrize("off", [2 ** 32, -(2 ** 32), 2 ** 40, 2 ** 62])
def test_paged(cuda_dev, n, L, off):
    assert _capi.device_error() == 0
    q = torch.randn(n, 4, 64, device=cuda_dev).bfloat16()
    pages = -(-L // 16)
    c = [torch.randn(pages, 16, 2, 64, device=cuda_dev).bfloat16() for _ in range(2)]
    args = dict(block_table=torch.arange(pages, device=cuda_dev)[None], kv_lens=torch.tensor([L], device=cuda_dev),
                cu_seqlens=torch.tensor([0, n], device=cuda_dev))
    want = bsk.attention_paged(q, *c, **{k: t.int() for k, t in args.items()})
    assert torch.equal(bsk.attention_paged(q, *c, **args), want)
    bsk.synchronize_and_check()
    for name, at in (("block_table", (0, 1)), ("kv_lens", 0), ("cu_seqlens", 1)):
        bad = {k: t.clone() for k, t in args.items()}
        bad[name][at] += off
        _reported(lambda: bsk.attention_paged(q, *c, **bad))
    assert _capi.device_error() == 0


def test_packed(cuda_dev):
    assert _capi.device_error() == 0
    q, k, v = (torch.randn(100, h, 64, device=cuda_dev).half() for h in (4, 2, 2))
    _reported(lambda: bsk.attention_varlen(q, k, v, torch.tensor([0, 60, 100 + 2 ** 32], device=cuda_dev)))
    _reported(lambda: bsk.attention_varlen(q, k, v, torch.tensor([0, 60 - 2 ** 32, 100], device=cuda_dev)))
    assert _capi.device_error() == 0
