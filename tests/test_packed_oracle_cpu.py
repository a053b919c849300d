"""The oracle's bound over e4m3 caches counts what the kernels round: weights in fp16, and no more."""
import torch

from oracle import packed_attention as pa


def _case(dtype, sizes=1.0):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(40, 2, 64, generator=g).to(dtype)
    k, v = torch.randn(4, 16, 1, 64, generator=g), torch.randn(4, 16, 1, 64, generator=g)
    v *= torch.as_tensor(sizes)
    (kc, ks), (vc, vs) = pa.quantise_rows(k), pa.quantise_rows(v)
    table = torch.tensor([[2, 0, 3, 1]])
    args = (q, kc, vc, table, [60], [40], 0.125, ks, vs)
    codes, s = vc[table[0]].flatten(0, 1)[:60, 0].double(), vs[table[0]].flatten(0, 1)[:60, 0].double()
    keys = (kc[table[0]].flatten(0, 1).double() * ks[table[0]].flatten(0, 1).double()[..., None])[:60, 0]
    allowed = torch.arange(60) <= 20 + torch.arange(40)[:, None]
    p = [torch.softmax((q[:, h].double() @ keys.t() * 0.125).masked_fill(~allowed, float("-inf")), -1) for h in range(2)]
    return args, p, s, codes, allowed


def _rounded(p, s, codes, weights, dtype, unit):
    """O from weights P * s / unit, rounded by `weights`."""
    return torch.stack([(weights(ph * s / unit(ph)).double() @ codes * unit(ph)).to(dtype) for ph in p], 1)


def test_fp16_weights_are_within_and_bf16_weights_are_not():
    args, p, s, codes, allowed = _case(torch.float16)
    want = pa.paged64(*args)
    for unit in (lambda ph: (ph * s).amax(-1, keepdim=True), lambda ph: (allowed * s).amax(-1, keepdim=True)):
        assert pa.worst(_rounded(p, s, codes, torch.Tensor.half, torch.float16, unit), *want) <= 1.0
        assert pa.worst(_rounded(p, s, codes, torch.Tensor.bfloat16, torch.float16, unit), *want) > 1.0


def test_values_of_very_different_sizes():
    """Subnormal fp16 weights are within the bound; weights below fp16's range altogether, by another reference, are not."""
    sizes = torch.exp2(-torch.arange(64).view(4, 16, 1, 1).float() / 2)  # down to 2^-31.5 of the largest
    args, p, s, codes, allowed = _case(torch.bfloat16, sizes)
    want = pa.paged64(*args)
    own = lambda ph: (allowed * s).amax(-1, keepdim=True) * 2.0 ** -6  # noqa: E731
    assert pa.worst(_rounded(p, s, codes, torch.Tensor.half, torch.bfloat16, own), *want) <= 1.0
    foreign = lambda ph: s.amax() * 2.0 ** 30 + 0 * own(ph)  # noqa: E731
    assert pa.worst(_rounded(p, s, codes, torch.Tensor.half, torch.bfloat16, foreign), *want) > 1.0
