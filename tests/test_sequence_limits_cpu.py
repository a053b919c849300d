"""More sequences than the kernels' 32-bit counters step through are refused through the C ABI; the largest number passes the
checks."""
import pytest
import torch

from periodicdent42_b200 import _capi

BUF = torch.zeros(4096, dtype=torch.uint8)
P = (BUF.data_ptr() + 15) // 16 * 16
BIG = 1 << 62
MOST = 2 ** 31 - 2 ** 17 - 1


def _plan(batch):
    return _capi.lib().bsk_kv_cache_plan(P, P, batch, P, 4, 4, P, 4, P, 16, P, P, 3, P, P, P, None)


def _paged(batch, window):
    name, more = ("bsk_attention_paged_window", (4, 1)) if window else ("bsk_attention_paged", ())
    return getattr(_capi.lib(), name)(0, P, 64, 64, P, P, 0, None, None, P, 2, 2, P, P, P, 1, batch, 2, 1, 64, 2, 16, 0.1, *more, P, BIG, None)


def _forward(batch, window, kv_heads=1):
    name, more = ("bsk_attention_varlen_window_fwd", (4, 1)) if window else ("bsk_attention_varlen_fwd", (1,))
    return getattr(_capi.lib(), name)(0, P, 64, 64, P, 64, 64, P, 64, 64, P, P, None, 1, batch, kv_heads, kv_heads, 64, 0.1,
                                      *more, P, BIG, None)


def _backward(batch, window, kv_heads=1):
    name, more = ("bsk_attention_varlen_window_bwd", (4, 1)) if window else ("bsk_attention_varlen_bwd", (1,))
    return getattr(_capi.lib(), name)(0, P, 64, 64, P, 64, 64, P, 64, 64, P, 64, 64, P, P, P, P, P, P, 1, batch, kv_heads, kv_heads, 64,
                                      0.1, *more, P, BIG, None)


CALLS = [_plan] + [lambda b, f=f, w=w: f(b, w) for f in (_paged, _forward, _backward) for w in (False, True)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("batch", [MOST + 1, 2 ** 31 - 513, 2 ** 31 - 1])
def test_more_are_refused(call, batch):
    assert call(batch) == _capi.BSK_ERR_UNSUPPORTED, _capi.last_error()


@pytest.mark.parametrize("window", [False, True])
def test_items_of_all_kv_heads_count(window):
    for call in (_forward, _backward):
        assert call(MOST // 8, window, 8) == _capi.BSK_ERR_UNSUPPORTED and "too many" in _capi.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch")
@pytest.mark.parametrize("call", CALLS)
def test_largest_is_taken(call):
    for batch in (1, MOST - 2):  # (a tile and an empty slot beside the sequences)
        assert call(batch) == _capi.BSK_ERR_NO_DEVICE, _capi.last_error()
