"""Rotary, cache and packed / paged attention without a GPU: refusals through the C ABI and the public functions, rotary
frequencies, and the oracle against torch's autograd."""
import math

import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi


def _rc(name, *args):
    rc = getattr(_capi.lib(), name)(*args)
    return rc, _capi.last_error()


BUF = torch.zeros(4096, dtype=torch.uint8)
P = (BUF.data_ptr() + 15) // 16 * 16


def _rotary(**kw):
    a = dict(dtype=0, Q=P, q_ts=64, q_hs=64, Qo=P, heads=1, K=P, k_ts=64, k_hs=64, Ko=P, kv_heads=1, pos=P, pos_bytes=8, freq=P,
             tokens=1, dim=64, r=64, inter=0, scale=1.0, backward=0, stream=None)
    a.update(kw)
    return _rc("bsk_rotary", *a.values())


@pytest.mark.parametrize("change", [dict(dtype=3), dict(tokens=-1), dict(r=63), dict(r=66), dict(r=0), dict(pos_bytes=2),
                                    dict(scale=float("nan")), dict(scale=float("inf")), dict(pos=None), dict(Qo=None), dict(K=None)])
def test_rotary_arguments(change):
    assert _rotary(**change)[0] == _capi.BSK_ERR_INVALID_ARG


@pytest.mark.parametrize("dim", [0, 63, 514])
def test_rotary_head_dim(dim):
    assert _rotary(dim=dim, r=2)[0] == _capi.BSK_ERR_UNSUPPORTED


def _append(**kw):
    a = dict(dtype=0, K=P, k_ts=64, k_hs=64, V=P, v_ts=64, v_hs=64, kc=P, vc=P, e4m3=0, ks=None, vs=None, slots=P, slot_bytes=8,
             tokens=1, heads=1, dim=64, num=8, stream=None)
    a.update(kw)
    return _rc("bsk_kv_cache_append", *a.values())[0]


def test_cache_arguments():
    for change in (dict(dtype=2), dict(tokens=-1), dict(slot_bytes=1), dict(K=None), dict(K=P + 2), dict(k_ts=36), dict(v_hs=4),
                   dict(kc=None), dict(vc=P + 8), dict(e4m3=1), dict(num=-1), dict(slots=None)):
        assert _append(**change) == _capi.BSK_ERR_INVALID_ARG, change
    for change in (dict(dim=32), dict(dim=256), dict(tokens=2 ** 30, heads=4)):
        assert _append(**change) == _capi.BSK_ERR_UNSUPPORTED, change
    gather = [0, P, P, 0, None, None, P, 8, P, P, 1, 1, 64, 8, None]
    for i, x, code in ((0, 2, -1), (8, None, -1), (9, P + 4, -1), (12, 96, -2), (3, 1, -1)):
        bad = list(gather)
        bad[i] = x
        assert _rc("bsk_kv_cache_gather", *bad)[0] == code


def _paged(**kw):
    a = dict(dtype=0, Q=P, q_ts=64, q_hs=64, kc=P, vc=P, e4m3=0, ks=None, vs=None, table=P, ts=2, width=2, lens=P, cu=P, O=P, tokens=1,
             batch=1, heads=2, kv_heads=1, dim=64, pages=2, page=16, scale=0.1, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _rc("bsk_attention_paged", *a.values())[0]


def test_paged_arguments():
    for change in (dict(dtype=2), dict(tokens=-1), dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(heads=0), dict(scale=0.0),
                   dict(scale=float("nan")), dict(Q=None), dict(table=None), dict(lens=None), dict(cu=None), dict(O=P + 2),
                   dict(q_ts=60), dict(e4m3=1), dict(pages=-1)):
        assert _paged(**change) == _capi.BSK_ERR_INVALID_ARG, change
    for change in (dict(dim=96), dict(page=4), dict(page=24), dict(page=2048), dict(heads=129), dict(pages=2 ** 28, page=16),
                   dict(width=2 ** 28, page=16)):
        assert _paged(**change) == _capi.BSK_ERR_UNSUPPORTED, change


def test_varlen_arguments():
    ws = _capi.lib().bsk_attention_varlen_workspace_bytes
    assert ws(100, 2, 8, 2, 64, 0) >= 0 and ws(100, 2, 8, 2, 64, 1) >= 0
    assert ws(100, 2, 8, 3, 64, 0) == _capi.BSK_ERR_INVALID_ARG and ws(100, 2, 8, 2, 80, 0) == _capi.BSK_ERR_UNSUPPORTED
    big = 1 << 40
    fwd = [0, P, 64, 64, P, 64, 64, P, 64, 64, P, P, None, 1, 1, 1, 1, 64, 0.1, 1, P, big, None]
    for i, x, code in ((0, 7, -1), (1, None, -1), (4, P + 2, -1), (8, 12, -1), (11, None, -1), (13, -1, -1), (16, 0, -1), (17, 32, -2),
                       (18, -1.0, -1), (20, P + 8, -1)):
        bad = list(fwd)
        bad[i] = x
        assert _rc("bsk_attention_varlen_fwd", *bad)[0] == code, i
    bwd = [0] + [P, 64, 64] * 4 + [P, P, P, P, P, P, 1, 1, 1, 1, 64, 0.1, 1, P, big, None]
    for i, x, code in ((1, None, -1), (2, 4, -1), (13, None, -1), (14, None, -1), (16, P + 2, -1), (18, None, -1), (23, 100, -2)):
        bad = list(bwd)
        bad[i] = x
        assert _rc("bsk_attention_varlen_bwd", *bad)[0] == code, i


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_no_device_fails_loudly():
    assert _rotary()[0] == _append() == _paged() == _capi.BSK_ERR_NO_DEVICE


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    i = torch.arange(4)
    for call in (lambda: bsk.rotary_embedding(q, k, i, torch.ones(32)), lambda: bsk.kv_cache_append(k, k, c, c, i),
                 lambda: bsk.kv_cache_gather(c, c, i), lambda: bsk.attention_varlen(q, k, k, i.int()),
                 lambda: bsk.attention_varlen(q.requires_grad_(True), k, k, i.int()),
                 lambda: bsk.attention_paged(q.detach(), c, c, i[None].int(), i[:1].int(), i[:2].int())):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="dtype"):
        bsk.kv_cache_gather(c, c, i, dtype=torch.float32)


def test_rotary_frequencies():
    f, s = bsk.rotary_frequencies(8, 10000.0)
    assert s == 1.0 and f.dtype == torch.float32
    assert torch.allclose(f.double(), torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=2 ** -23)
    assert torch.allclose(bsk.rotary_frequencies(8, scaling="linear", factor=4)[0], f / 4)
    ntk = bsk.rotary_frequencies(8, scaling="ntk", factor=4)[0]
    assert ntk[0] == 1 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-6)
    y, s = bsk.rotary_frequencies(128, scaling="yarn", factor=8, original_length=4096)
    base = bsk.rotary_frequencies(128)[0]
    assert math.isclose(s, 0.1 * math.log(8) + 1)
    turns = 4096 * base.double() / (2 * math.pi)
    assert torch.equal(y[turns > 40], base[turns > 40])          # fast pairs kept
    slow = turns < 0.7
    assert slow.any() and torch.allclose(y[slow], base[slow] / 8)  # slow pairs divided
    ratio = (y / base).double()
    assert (ratio[1:] <= ratio[:-1] + 1e-7).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, base=-1.0),
                dict(rotary_dim=8, scaling="linear", factor=0.5), dict(rotary_dim=2, scaling="ntk", factor=2),
                dict(rotary_dim=8, scaling="yarn", factor=2, beta_fast=1, beta_slow=2)):
        with pytest.raises(ValueError):
            bsk.rotary_frequencies(**bad)


def test_oracle_gradients_match_autograd():
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(n, 16, generator=g, dtype=torch.float64) for n in (9, 9, 9, 9))
    allowed = torch.ones(9, 9, dtype=torch.bool).tril()
    want = [t.clone().requires_grad_(True) for t in (q, k, v)]
    s = (want[0] @ want[1].t() * 0.25).masked_fill(~allowed, -math.inf).softmax(-1)
    o = s @ want[2]
    grads = torch.autograd.grad(o, want, do)
    got = pa.gradients64(q, k, v, do, allowed, 0.25, torch.bfloat16)
    assert torch.allclose(got["O"][0], o.detach())
    for n, w in zip(("dQ", "dK", "dV"), grads):
        assert torch.allclose(got[n][0], w, atol=1e-12)


def test_oracle_rounding_bound_holds_for_rounded_arithmetic():
    """Rounding P and O to 16 bits, as the kernels do, stays within the bound; a mistake planted in one key does not."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(40, 64, generator=g).bfloat16() for _ in range(3))
    allowed = torch.ones(40, 40, dtype=torch.bool).tril()
    o, bound, p, _, _ = pa.attention64(q, k, v, allowed, 0.125, torch.bfloat16)
    rounded = (p.bfloat16().double() @ v.double()).bfloat16()
    assert pa.worst(rounded, o, bound) <= 1.0
    v2 = v.clone()
    v2[3] = -v2[3]
    assert pa.worst(p @ v2.double(), o, bound) > 1.0


def test_quantise_rows_is_within_half_a_step():
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(2)).half()
    x[0] = 0
    c, s = pa.quantise_rows(x)
    back = c.double() * s.double()[:, None]
    # half a step of e4m3: 2^-4 relative, 2^-10 absolute below its normal range, both in units of the scale; two divisions' 2^-24
    assert ((back - x.double()).abs() <= x.double().abs() * (2.0 ** -4 + 2.0 ** -22) + s.double()[:, None] * 2.0 ** -10).all()
    assert s[0] == 0 and (back[0] == 0).all()
