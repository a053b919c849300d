"""Sizes that the paged kernels' 32-bit positions cannot hold are refused through the C ABI; the largest ones pass the checks."""
import pytest
import torch

from periodicdent42_b200 import _capi

BUF = torch.zeros(4096, dtype=torch.uint8)
P = (BUF.data_ptr() + 15) // 16 * 16
MOST = 2 ** 31 - 4096


def _paged(pages, width, page):
    return _capi.lib().bsk_attention_paged(0, P, 64, 64, P, P, 0, None, None, P, width, width, P, P, P, 1, 1, 2, 1, 64, pages, page,
                                           0.1, P, 1 << 40, None)


@pytest.mark.parametrize("page", [8, 16, 128, 1024])
def test_largest_and_next(page):
    for pages, width in ((MOST // page + 1, 1), (1, MOST // page + 1), ((2 ** 31 - 8) // page, 1), (1, (2 ** 31 - 8) // page)):
        if max(pages, width) * page > MOST:
            assert _paged(pages, width, page) == _capi.BSK_ERR_UNSUPPORTED
            assert "2^31 - 4096" in _capi.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch")
@pytest.mark.parametrize("page", [8, 16, 128, 1024])
def test_largest_is_taken(page):
    assert _paged(MOST // page, MOST // page, page) == _capi.BSK_ERR_NO_DEVICE
