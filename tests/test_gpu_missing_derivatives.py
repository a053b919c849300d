"""Derivatives that the decoder operators do not have are refused, not dropped: forward-mode tangents of all of them, gradients
of the ones for serving."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import periodicdent42_b200 as bsk

pytestmark = pytest.mark.gpu


def _calls(dev):
    q, k, v = (torch.randn(8, h, 64, device=dev).bfloat16() for h in (4, 2, 2))
    cache = [torch.randn(2, 16, 2, 64, device=dev).bfloat16() for _ in range(2)]
    codes = [torch.zeros(2, 16, 2, 64, device=dev).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(2, 16, 2, device=dev) for _ in range(2)]
    slots, pos = torch.arange(8, device=dev), torch.arange(8, device=dev)
    at = (torch.tensor([[0, 1]], device=dev), torch.tensor([20], device=dev), torch.tensor([0, 8], device=dev))
    freq = bsk.rotary_frequencies(64, device=dev)[0]
    return {
        "rotary": (lambda q, k: bsk.rotary_embedding(q, k, pos, freq), (q, k)),
        "varlen": (lambda q, k, v: bsk.attention_varlen(q, k, v, at[2]), (q, k, v)),
        "append": (lambda k, v, a, b: bsk.kv_cache_append(k, v, a, b, slots), (k, v, *cache)),
        "append e4m3": (lambda k, s: bsk.kv_cache_append(k, v, *codes, slots, s, scales[1]), (k, scales[0])),
        "gather": (lambda a, b: bsk.kv_cache_gather(a, b, slots), tuple(cache)),
        "paged": (lambda q, a, b: bsk.attention_paged(q, a, b, *at), (q, *cache)),
        "paged e4m3": (lambda q, s: bsk.attention_paged(q, *codes, *at, k_scale=scales[0], v_scale=s), (q, scales[1])),
    }


@pytest.mark.parametrize("name", ["rotary", "varlen", "append", "append e4m3", "gather", "paged", "paged e4m3"])
def test_tangents_are_refused(no_device_error, cuda_dev, name):
    call, args = _calls(cuda_dev)[name]
    call(*args)
    for i in range(len(args)):
        with fwd.dual_level():
            dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)


@pytest.mark.parametrize("name", ["append", "append e4m3", "gather", "paged", "paged e4m3"])
def test_gradients_of_the_serving_operators_are_refused(no_device_error, cuda_dev, name):
    call, args = _calls(cuda_dev)[name]
    for i in range(len(args)):
        needs = [t.clone().requires_grad_(True) if j == i else t for j, t in enumerate(args)]
        with pytest.raises(ValueError, match="no gradient"):
            call(*needs)
        with torch.no_grad():
            call(*needs)
        with torch.inference_mode():
            call(*needs)
