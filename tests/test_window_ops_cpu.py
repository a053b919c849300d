"""Windowed attention, norm with rotation, rotary axes and the plan of a serving step without a GPU: refusals through the C ABI
and the public functions, the axes' order, and the oracle against torch's autograd and loops."""
import math

import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

BUF = torch.zeros(4096, dtype=torch.uint8)
P = (BUF.data_ptr() + 15) // 16 * 16
INVALID, UNSUPPORTED = _capi.BSK_ERR_INVALID_ARG, _capi.BSK_ERR_UNSUPPORTED
BIG = 1 << 40


def _rc(name, args):
    return getattr(_capi.lib(), name)(*args.values())


def _paged(**kw):
    return _rc("bsk_attention_paged_window", {**dict(
        dtype=0, Q=P, q_ts=64, q_hs=64, kc=P, vc=P, e4m3=0, ks=None, vs=None, table=P, ts=2, width=2, lens=P, cu=P, O=P, tokens=1,
        batch=1, heads=2, kv_heads=1, dim=64, pages=2, page=16, scale=0.1, window=4, sinks=1, ws=P, ws_bytes=BIG, stream=None), **kw})


def _varlen(**kw):
    return _rc("bsk_attention_varlen_window_fwd", {**dict(
        dtype=0, Q=P, q_ts=64, q_hs=64, K=P, k_ts=64, k_hs=64, V=P, v_ts=64, v_hs=64, cu=P, O=P, lse=None, tokens=1, batch=1, heads=1,
        kv_heads=1, dim=64, scale=0.1, window=4, sinks=1, ws=P, ws_bytes=BIG, stream=None), **kw})


def _varlen_bwd(**kw):
    return _rc("bsk_attention_varlen_window_bwd", {**dict(
        dtype=0, dO=P, d_ts=64, d_hs=64, Q=P, q_ts=64, q_hs=64, K=P, k_ts=64, k_hs=64, V=P, v_ts=64, v_hs=64, O=P, lse=P, cu=P, dQ=P,
        dK=P, dV=P, tokens=1, batch=1, heads=1, kv_heads=1, dim=64, scale=0.1, window=4, sinks=1, ws=P, ws_bytes=BIG, stream=None), **kw})


def _norm(**kw):
    return _rc("bsk_qk_norm_rotary", {**dict(
        dtype=0, Q=P, q_ts=64, q_hs=64, Qo=P, heads=1, K=P, k_ts=64, k_hs=64, Ko=P, kv_heads=1, qw=P, kw=P, f32=0, pos=P, pos_bytes=8,
        axes=None, num_axes=1, freq=P, tokens=1, dim=64, r=64, inter=0, scale=1.0, eps=1e-6, stream=None), **kw})


def _norm_bwd(**kw):
    return _rc("bsk_qk_norm_rotary_bwd", {**dict(
        dtype=0, dQo=P, d_ts=64, d_hs=64, Q=P, q_ts=64, q_hs=64, dQ=P, heads=1, dKo=P, e_ts=64, e_hs=64, K=P, k_ts=64, k_hs=64, dK=P,
        kv_heads=1, qw=P, kw=P, f32=0, dqw=P, dkw=P, pos=P, pos_bytes=8, axes=None, num_axes=1, freq=P, tokens=1, dim=64, r=64, inter=0,
        scale=1.0, eps=1e-6, ws=P, ws_bytes=BIG, stream=None), **kw})


def _axes(**kw):
    return _rc("bsk_rotary_axes", {**dict(
        dtype=0, Q=P, q_ts=64, q_hs=64, Qo=P, heads=1, K=P, k_ts=64, k_hs=64, Ko=P, kv_heads=1, pos=P, pos_bytes=8, axes=P, num_axes=3,
        freq=P, tokens=1, dim=64, r=64, inter=0, scale=1.0, backward=0, stream=None), **kw})


def _plan(**kw):
    return _rc("bsk_kv_cache_plan", {**dict(
        kv=P, new=P, batch=2, table=P, stride=4, width=4, free=P, num_free=4, count=P, page=16, slots=P, pos=P, tokens=3, cu=P, lens=P,
        left=P, stream=None), **kw})


def test_window_arguments():
    for call in (_paged, _varlen, _varlen_bwd):
        for change in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(dtype=2), dict(tokens=-1), dict(heads=3, kv_heads=2),
                       dict(scale=0.0), dict(Q=None), dict(O=P + 2), dict(cu=None), dict(q_ts=60)):
            assert call(**change) == INVALID, change
        assert call(dim=96) == UNSUPPORTED
    assert _varlen(ws_bytes=0) == _varlen_bwd(ws_bytes=0) == INVALID
    ws = _capi.lib().bsk_attention_varlen_window_workspace_bytes
    assert ws(100, 2, 8, 2, 64, 0, 0, 0) == ws(100, 2, 8, 2, 64, 4, -1, 1) == ws(100, 2, 8, 3, 64, 4, 0, 0) == INVALID
    assert ws(100, 2, 8, 2, 64, 4, 0, 1) == _capi.lib().bsk_attention_varlen_workspace_bytes(100, 2, 8, 2, 64, 1)


def test_norm_axes_and_plan_arguments():
    for call in (_norm, _norm_bwd, _axes):
        for change in (dict(dtype=3), dict(tokens=-1), dict(r=63), dict(r=66), dict(pos_bytes=2), dict(scale=float("nan")), dict(pos=None),
                       dict(Q=None), dict(K=None), dict(freq=None), dict(axes=P, num_axes=0)):
            assert call(**change) == INVALID, change
        assert call(dim=514) == UNSUPPORTED
    assert _axes(axes=None) == INVALID
    for call in (_norm, _norm_bwd):
        for change in (dict(eps=0.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(qw=None), dict(kw=None)):
            assert call(**change) == INVALID, change
    assert _norm_bwd(dQo=None) == INVALID and _norm_bwd(dK=None) == INVALID
    for change in (dict(batch=-1), dict(tokens=-1), dict(width=-1), dict(num_free=-1), dict(page=0), dict(stride=3), dict(kv=None),
                   dict(table=None), dict(free=None), dict(count=None), dict(slots=None), dict(cu=None), dict(left=None)):
        assert _plan(**change) == INVALID, change


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_no_device_fails_loudly():
    for call in (_paged, _varlen, _varlen_bwd, _norm, _norm_bwd, _axes, _plan):
        assert call() == _capi.BSK_ERR_NO_DEVICE


def test_cpu_tensors_and_bad_windows_are_refused():
    q, k, w = torch.zeros(4, 2, 64).bfloat16(), torch.zeros(4, 1, 64).bfloat16(), torch.ones(64).bfloat16()
    c, i = torch.zeros(1, 16, 1, 64).bfloat16(), torch.arange(4)
    for call in (lambda: bsk.qk_norm_rotary(q, k, w, w, i, torch.ones(32)),
                 lambda: bsk.rotary_embedding(q, k, i[None], torch.ones(32), axes=torch.zeros(32, dtype=torch.int32)),
                 lambda: bsk.attention_varlen(q, k, k, i.int(), window=2), lambda: bsk.kv_cache_plan(i, i, i[None].int(), i, i, 16, 4),
                 lambda: bsk.attention_paged(q, c, c, i[None].int(), i[:1].int(), i[:2].int(), window=2, sinks=1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for kw in (dict(window=0), dict(window=-2)):
        with pytest.raises(ValueError, match="window"):
            bsk.attention_varlen(q, k, k, i.int(), **kw)


def test_rotary_axes():
    assert bsk.rotary_axes((2, 1, 3)).tolist() == [0, 0, 1, 2, 2, 2] and bsk.rotary_axes((2, 1, 3)).dtype == torch.int32
    assert bsk.rotary_axes((2, 1, 3), cycle=True).tolist() == [0, 1, 2, 0, 2, 2]
    assert bsk.rotary_axes((0, 2), cycle=True).tolist() == [1, 1] and bsk.rotary_axes([3]).tolist() == [0, 0, 0]
    a = bsk.rotary_axes((24, 20, 20), cycle=True)
    assert a[:60].tolist() == [0, 1, 2] * 20 and a[60:].tolist() == [0] * 4
    for bad in ((), (0, 0), (3, -1)):
        with pytest.raises(ValueError):
            bsk.rotary_axes(bad)


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (100, 0), (2, 100), (None, 0)])
def test_visible_keys_one_by_one(window, sinks):
    place = torch.tensor([-1, 0, 1, 4, 9, 20])
    got = pa.visible(place, 12, window, sinks)
    for r, p in enumerate(place.tolist()):
        for j in range(12):
            assert bool(got[r, j]) == (j <= p and (window is None or j > p - window or j < sinks))


def test_norm_oracle_matches_autograd():
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(7, 3, 16, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.rand(16, generator=g, dtype=torch.float64) + 0.5
    pos, f = torch.randint(0, 50, (3, 7), generator=g), bsk.rotary_frequencies(12)[0]
    axes = bsk.rotary_axes((2, 3, 1), cycle=True)
    for inter in (False, True):
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        z = xs / (xs.square().mean(-1, keepdim=True) + 1e-3).sqrt() * ws
        angle = torch.stack([pos[a].double() * q for a, q in zip(axes.tolist(), f.double().tolist())], 1)[:, None]
        a, b = (z[..., 0:12:2], z[..., 1:12:2]) if inter else (z[..., :6], z[..., 6:12])
        u, v = 1.3 * (a * angle.cos() - b * angle.sin()), 1.3 * (a * angle.sin() + b * angle.cos())
        y = torch.cat([torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1), z[..., 12:]], -1)
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
        got = pa.norm_rotary64(x, w, pos, f, inter, 1.3, 1e-3, axes, dy)
        for name, want in (("y", y.detach()), ("dx", dx), ("dw", dw)):
            assert torch.allclose(got[name][0], want, atol=1e-12), name


def test_norm_bound_holds_for_rounded_arithmetic():
    """The formulas in fp32, rounded once, stay within the bound; a weight that is off by a rounding step of bf16 does not."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(30, 2, 64, generator=g).bfloat16()
    w, pos, f = (torch.rand(64, generator=g) + 0.5), torch.arange(30), bsk.rotary_frequencies(64)[0]

    def run(weight):
        y = x.float()
        z = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight
        return pa.rotary64(z, pos, f, False, 1.0).float().bfloat16()

    want = pa.norm_rotary64(x, w, pos, f, False, 1.0, 1e-6)["y"]
    assert pa.worst(run(w), *want) <= 1.0
    assert pa.worst(run(w * (1 + 2.0 ** -6)), *want) > 1.0


def test_plan_oracle():
    slots, places, cu, lens, stack, table = pa.plan_steps([3, 0, 4], [2, 0, 1], [[5, -1], [-1, -1], [2, -1]], [9, 8, 7], 4, 5)
    assert slots == [23, 28, 32, -1, -1] and places == [3, 4, 4, 0, 0] and cu == [0, 2, 2, 3] and lens == [5, 0, 5]
    assert stack == [9] and table == [[5, 7], [-1, -1], [2, 8]]
    assert math.isclose(pa._norm_error(64), (33.5 + 4) * 2.0 ** -24)
