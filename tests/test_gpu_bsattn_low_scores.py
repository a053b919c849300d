"""Block-sparse attention where every score of a row is far below zero (or far above): the row's maximum is that of its own
scores and of nothing else. Elementwise within the bound of oracle/packed_attention.py: weights are rounded to 16 bits (half a
step, 2^-8 in bf16, of each P_j |v_j|), and all rows here have the same few large weights, so that these roundings do not
average out; a normwise 1e-3 has no room for them."""
import pytest
import torch

from oracle import packed_attention as pa
from periodicdent42_b200 import _capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 128), (torch.float16, 64)])
def test_scores_far_from_zero(no_device_error, cuda_dev, dtype, D, causal, sign):
    g = torch.Generator().manual_seed(D)
    S, nqb = 384, 3
    q = torch.full((1, 1, S, D), 8.0)
    k = sign * (8.0 + torch.randn(1, 1, S, D, generator=g) / 4)
    q, k, v = (t.to(dtype) for t in (q, k, torch.randn(1, 1, S, D, generator=g)))
    cols = [list(range(i + 1)) if causal else list(range(nqb)) for i in range(nqb)]
    rp = torch.tensor([0] + [len(c) for c in cols]).cumsum(0).int()
    ci = torch.tensor([j for c in cols for j in c]).int()
    scale = D ** -0.5
    O = torch.full_like(q, float("nan"), device=cuda_dev)
    lse = torch.empty(S, device=cuda_dev)
    _capi.bsattn_fwd_ex(*(t.to(cuda_dev) for t in (q, k, v)), O, lse, rp.to(cuda_dev), ci.to(cuda_dev), scale, causal)
    allowed = torch.ones(S, S, dtype=torch.bool)
    allowed = allowed.tril() if causal else allowed
    want, bound = pa.attention64(q[0, 0], k[0, 0], v[0, 0], allowed, scale, dtype)[:2]
    assert pa.worst(O.cpu()[0, 0], want, bound) <= 1.0
    s = q[0, 0].double() @ k[0, 0].double().t() * scale
    s = s.masked_fill(~allowed, float("-inf"))
    # fp32 sums of D products of about 64: (D + 8) 2^-24 of their size; the sum's exponentials 2.1e-4
    assert (lse.cpu().double() - torch.logsumexp(s, -1)).abs().max() <= (D + 8) * 2.0 ** -24 * 64 * D * scale * 1.2 + 2.1e-4
