"""The serving operators together, as a decoder uses them: rotary positions, the cache written chunk by chunk, attention of
each chunk over it, single tokens at the end -- against attention over the whole packed sequences."""
import pytest
import torch

import periodicdent42_b200 as bsk
from oracle import packed_attention as pa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype,H,G,D,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 6, 6, 64, 64)])
def test_chunks_then_single_tokens(no_device_error, cuda_dev, e4m3, dtype, H, G, D, page):
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    lens = [150, 41, 203]
    T, B = sum(lens), len(lens)
    start = [0, 150, 191]
    q, k, v = (torch.randn(T, n, D, generator=g, device=cuda_dev).to(dtype) for n in (H, G, G))
    pos = torch.cat([torch.arange(n, device=cuda_dev) for n in lens])
    inv_freq, scale = bsk.rotary_frequencies(D, scaling="yarn", factor=4.0, original_length=64, device=cuda_dev)
    width = -(-max(lens) // page)
    pages = B * width
    table = torch.randperm(pages, generator=g, device=cuda_dev).int().view(B, width)
    shape = (pages, page, G, D)
    kind = torch.float8_e4m3fn if e4m3 else dtype
    c = dict(k_cache=torch.empty(shape, device=cuda_dev, dtype=kind), v_cache=torch.empty(shape, device=cuda_dev, dtype=kind))
    if e4m3:
        c.update(k_scale=torch.empty(shape[:3], device=cuda_dev), v_scale=torch.empty(shape[:3], device=cuda_dev))
    outs = [[] for _ in range(B)]
    done = [0] * B
    for step in [(100, 7, 128), (49, 33, 74), (1, 1, 1)]:
        rows = torch.cat([torch.arange(s + d, s + d + n, device=cuda_dev) for s, d, n in zip(start, done, step)])
        seq = torch.repeat_interleave(torch.arange(B, device=cuda_dev), torch.tensor(step, device=cuda_dev))
        p = pos[rows]
        slots = table[seq, (p // page)].long() * page + p % page
        qr, kr = bsk.rotary_embedding(q[rows], k[rows], p, inv_freq, scale=scale)
        bsk.kv_cache_append(kr, v[rows], slots=slots, **c)
        done = [d + n for d, n in zip(done, step)]
        cu = torch.tensor([0, *step], device=cuda_dev).cumsum(0)
        o = bsk.attention_paged(qr, block_table=table, kv_lens=torch.tensor(done, device=cuda_dev), cu_seqlens=cu, **c)
        for i, part in enumerate(o.split(list(step))):
            outs[i].append(part)
    got = torch.cat([torch.cat(parts) for parts in outs])
    assert done == lens
    qa, ka = bsk.rotary_embedding(q, k, pos, inv_freq, scale=scale)
    cu = torch.tensor([0, *lens], device=cuda_dev).cumsum(0).int()
    if not e4m3:
        # both kernels are within the definition's bound of the same definition
        want = pa.packed64(qa, ka, v, lens, True, D ** -0.5)["O"]
        assert pa.worst(got, *want) <= 1.0
        assert pa.worst(bsk.attention_varlen(qa, ka, v, cu), *want) <= 1.0
        return
    # e4m3: what was written reads back as the quantised rows, and attention is the definition's on those rows
    seq = torch.repeat_interleave(torch.arange(B, device=cuda_dev), torch.tensor(lens, device=cuda_dev))
    slots = table[seq, pos // page].long() * page + pos % page
    codes, s = pa.quantise_rows(ka)
    assert torch.equal(bsk.kv_cache_gather(slots=slots, dtype=dtype, **c)[0], (codes.float() * s[..., None]).to(dtype))
    want = pa.paged64(qa, c["k_cache"], c["v_cache"], table, lens, lens, D ** -0.5, c["k_scale"], c["v_scale"])
    assert pa.worst(got, *want) <= 1.0


def test_training_step_through_rotary_and_packed_attention(no_device_error, cuda_dev):
    """Gradients through both operators together against torch's autograd of the 64-bit chain."""
    lens, H, G, D = [90, 47], 4, 2, 64
    T = sum(lens)
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    x = [torch.randn(T, n, D, generator=g, device=cuda_dev).half().requires_grad_(True) for n in (H, G, G)]
    do = torch.randn(T, H, D, generator=g, device=cuda_dev).half()
    pos = torch.cat([torch.arange(n, device=cuda_dev) for n in lens])
    f, _ = bsk.rotary_frequencies(D, device=cuda_dev)
    cu = torch.tensor([0, *lens], device=cuda_dev).cumsum(0).int()
    qr, kr = bsk.rotary_embedding(x[0], x[1], pos, f)
    got = torch.autograd.grad(bsk.attention_varlen(qr, kr, x[2], cu), x, do)
    y = [t.detach().double().requires_grad_(True) for t in x]

    def turn(t):
        angle = pos.double()[:, None] * f.double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = t[..., : D // 2], t[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    q64, k64, parts, a = turn(y[0]), turn(y[1]), [], 0
    for n in lens:
        r = slice(a, a + n)
        s = torch.einsum("qhd,khd->hqk", q64[r], k64[r].repeat_interleave(H // G, 1)) * D ** -0.5
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=cuda_dev).tril(), float("-inf"))
        parts.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), y[2][r].repeat_interleave(H // G, 1)))
        a += n
    want = torch.autograd.grad(torch.cat(parts), y, do.double())
    for a, b in zip(got, want):  # three fp16 roundings in a row (2^-11 each) on sums of many terms: 4 * 2^-11 normwise
        assert (a.double() - b).norm() <= 4 * 2.0 ** -11 * b.norm()
