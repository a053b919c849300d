"""The paged cache written and read back: bit-exact copies and codes, untouched slots, padding, bad slots, refusals."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


def _cache(pages, page, heads, dim, dtype, dev, e4m3):
    if not e4m3:
        k, v = (torch.randn(pages, page, heads, dim, device=dev).to(dtype) for _ in range(2))
        return dict(k_cache=k, v_cache=v)
    c = [torch.randint(0, 120, (pages, page, heads, dim), device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
         for _ in range(2)]
    s = [torch.rand(pages, page, heads, device=dev) for _ in range(2)]
    return dict(k_cache=c[0], v_cache=c[1], k_scale=s[0], v_scale=s[1])


def _bits(t):
    return t.view(torch.uint8)


def _same(a, b):
    return torch.equal(_bits(a.contiguous()), _bits(b.contiguous()))


def _expected(c, k, v, slots):
    c = {n: t.clone() for n, t in c.items()}
    keep = slots >= 0
    at, e4m3 = slots[keep].long(), "k_scale" in c
    for n, x in (("k", k[keep]), ("v", v[keep])):
        flat = _bits(c[n + "_cache"]).view(-1, x.shape[1] * x.shape[2] * c[n + "_cache"].element_size())
        if e4m3:
            x, s = pa.quantise_rows(x)
            c[n + "_scale"].view(-1, x.shape[1])[at] = s
        flat[at] = _bits(x.contiguous()).view(x.shape[0], -1)
    return c


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,heads,dim,page,pages", [(1, 1, 64, 8, 1), (17, 3, 128, 16, 3), (300, 8, 128, 64, 7), (65, 5, 64, 128, 2)])
def test_append_and_gather(no_device_error, cuda_dev, e4m3, dtype, T, heads, dim, page, pages):
    g = torch.Generator(device=cuda_dev).manual_seed(T)
    c = _cache(pages, page, heads, dim, dtype, cuda_dev, e4m3)
    k, v = (torch.randn(T, heads, dim, generator=g, device=cuda_dev).to(dtype) * 3 for _ in range(2))
    slots = torch.full((T,), -1, device=cuda_dev)
    n = min(T, pages * page)
    slots[:n] = torch.randperm(pages * page, generator=g, device=cuda_dev)[:n]
    slots = slots[torch.randperm(T, generator=g, device=cuda_dev)]
    if T > 4:
        slots[2] = -7  # padding inside the batch
    if heads > 1:  # rows of every size: zero, subnormal, the type's largest
        k[0, 0], k[0, 1], v[-1, 0] = 0, torch.finfo(dtype).tiny / 2, torch.finfo(dtype).max
    want = _expected(c, k, v, slots)
    for s in (slots, slots.int()):
        got = {n: t.clone() for n, t in c.items()}
        bsk.kv_cache_append(k, v, slots=s, **got)
        for name in c:
            assert _same(got[name], want[name]), name
    kr, vr = bsk.kv_cache_gather(slots=slots, dtype=dtype, **got)
    for r, x, n in ((kr, k, "k"), (vr, v, "v")):
        if e4m3:
            codes, scale = pa.quantise_rows(x)
            x = (codes.float() * scale[..., None]).to(dtype)
        assert _same(r, torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)))
    twice = torch.cat([slots, slots.flip(0)])  # reading a slot more than once is fine
    assert _same(bsk.kv_cache_gather(slots=twice, dtype=dtype, **got)[0], torch.cat([kr, kr.flip(0)]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_next_to_rounding_middles(no_device_error, cuda_dev, dtype):
    """Rows whose quotients lie on, just below and just above the middles between codes, in the normal and the subnormal
    range: every code is that of the IEEE quotient."""
    steps = torch.arange(16, dtype=torch.float64)
    mids = torch.cat([(1 + (2 * steps[:8] + 1) / 16)[None] * 2.0 ** e for e in torch.arange(-6, 9)[:, None]])
    subs = (2 * steps[:8] + 1) * 2.0 ** -10
    q = torch.cat([mids.flatten(), subs, 2.0 ** -6 + subs[:1]]).clamp(max=447)
    T = 4096
    g = torch.Generator().manual_seed(1)
    top = torch.rand(T, generator=g, dtype=torch.float64) * 4 + 0.01  # the rows' largest elements
    pick = torch.randint(0, q.numel(), (T, 128), generator=g)
    x = (q[pick] * top[:, None] / 448).to(dtype)
    x[:, 0] = top.to(dtype)
    x = (x * torch.where(torch.rand(T, 128, generator=g) < 0.5, -1, 1)).to(dtype)[:, None].contiguous().to(cuda_dev)
    c = _cache(64, 64, 1, 128, None, cuda_dev, True)
    want = _expected(c, x, x.flip(0), torch.arange(T, device=cuda_dev))
    bsk.kv_cache_append(x, x.flip(0), slots=torch.arange(T, device=cuda_dev), **c)
    assert all(_same(c[n], want[n]) for n in c)


@pytest.mark.parametrize("other", [torch.bfloat16, torch.float16])
def test_gather_of_codes_in_either_type(no_device_error, cuda_dev, other):
    c = _cache(3, 16, 2, 64, None, cuda_dev, True)
    slots = torch.arange(48, device=cuda_dev)
    k, _ = bsk.kv_cache_gather(slots=slots, dtype=other, **c)
    assert _same(k, (c["k_cache"].float() * c["k_scale"][..., None]).to(other).view(48, 2, 64))


def test_non_finite_rows_mark_their_row_only(no_device_error, cuda_dev):
    c = _cache(1, 16, 2, 64, torch.bfloat16, cuda_dev, True)
    k = torch.randn(3, 2, 64, device=cuda_dev).bfloat16()
    k[0, 0, 5], k[1, 1, 63] = float("nan"), float("inf")
    slots = torch.tensor([3, 0, 9], device=cuda_dev)
    bsk.kv_cache_append(k, k.clone(), slots=slots, **c)
    r, _ = bsk.kv_cache_gather(slots=slots, dtype=torch.bfloat16, **c)
    bad = torch.zeros(3, 2, dtype=torch.bool, device=cuda_dev)
    bad[0, 0] = bad[1, 1] = True
    assert torch.equal(torch.isnan(r).any(-1), bad)
    assert torch.isnan(r[0, 0]).all()


def test_strided_rows(no_device_error, cuda_dev):
    x = torch.randn(40, 12, 128, device=cuda_dev).half()
    k, v = x[:, 4:8], x[:, 8:]
    c = _cache(2, 32, 4, 128, torch.float16, cuda_dev, False)
    slots = torch.arange(40, device=cuda_dev) + 11
    want = _expected(c, k, v, slots)
    version = c["k_cache"]._version
    bsk.kv_cache_append(k, v, slots=slots, **c)
    assert _same(c["k_cache"], want["k_cache"]) and _same(c["v_cache"], want["v_cache"])
    assert c["k_cache"]._version > version  # autograd sees the write
    c2 = {n: t.clone() for n, t in c.items()}
    odd = torch.randn(40 * 4 * 128 + 3, device=cuda_dev).half()[3:].view(40, 4, 128)
    bsk.kv_cache_append(odd, k.transpose(0, 1).contiguous().transpose(0, 1), slots=slots, **c2)
    want = _expected(c, odd, k, slots)
    assert _same(c2["k_cache"], want["k_cache"]) and _same(c2["v_cache"], want["v_cache"])


def test_slot_behind_the_cache_is_reported(cuda_dev):
    assert _capi.device_error() == 0
    c = _cache(2, 8, 1, 64, torch.bfloat16, cuda_dev, False)
    before = {n: t.clone() for n, t in c.items()}
    k = torch.randn(2, 1, 64, device=cuda_dev).bfloat16()
    bsk.kv_cache_append(k, k, slots=torch.tensor([16, -1], device=cuda_dev), **c)
    with pytest.raises(RuntimeError, match="out-of-range"):
        bsk.synchronize_and_check()
    assert all(_same(c[n], before[n]) for n in c)
    r, _ = bsk.kv_cache_gather(slots=torch.tensor([2 ** 40, 3], device=cuda_dev), **c)
    with pytest.raises(RuntimeError, match="out-of-range"):
        bsk.synchronize_and_check()
    assert (r[0] == 0).all() and _same(r[1], c["k_cache"].view(16, 1, 64)[3])
    assert _capi.device_error() == 0


def test_refusals(cuda_dev):
    c, q = _cache(2, 8, 2, 64, torch.bfloat16, cuda_dev, False), _cache(2, 8, 2, 64, None, cuda_dev, True)
    k = torch.randn(3, 2, 64, device=cuda_dev).bfloat16()
    slots = torch.arange(3, device=cuda_dev)
    base = dict(K=k, V=k, slots=slots, **c)
    bad = [dict(K=k[0]), dict(V=k[:2]), dict(K=k.float(), V=k.float()), dict(K=k.half(), V=k.half()), dict(V=k.half()),
           dict(K=k.cpu()), dict(slots=slots[:2]), dict(slots=slots.float()), dict(slots=slots.cpu()), dict(slots=slots[None]),
           dict(K=k[:, :1], V=k[:, :1]), dict(k_cache=c["k_cache"].transpose(0, 1)), dict(k_cache=c["k_cache"][:1]),
           dict(k_scale=q["k_scale"]), dict(k_scale=q["k_scale"], v_scale=q["v_scale"]), dict(k_cache=q["k_cache"]),
           dict(k_cache=q["k_cache"], v_cache=q["v_cache"]),
           dict(k_cache=q["k_cache"], v_cache=q["v_cache"], k_scale=q["k_scale"], v_scale=q["v_scale"].double()),
           dict(k_cache=q["k_cache"], v_cache=q["v_cache"], k_scale=q["k_scale"], v_scale=q["v_scale"][:1])]
    for change in bad:
        with pytest.raises(ValueError):
            bsk.kv_cache_append(**{**base, **change})
    with pytest.raises(ValueError):
        bsk.kv_cache_append(k[..., :32], k[..., :32], c["k_cache"][..., :32].contiguous(), c["v_cache"][..., :32].contiguous(), slots)
    for dtype in (torch.float16, torch.float32):
        with pytest.raises(ValueError):
            bsk.kv_cache_gather(slots=slots, dtype=dtype, **c)
    bsk.kv_cache_append(k[:0], k[:0], slots=slots[:0], **c)  # no tokens is no error
    assert bsk.kv_cache_gather(slots=slots[:0], **c)[0].shape == (0, 2, 64)
