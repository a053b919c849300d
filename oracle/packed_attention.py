"""64-bit definitions of rotary positions, the quantised cache and attention over packed or cached sequences, with
elementwise bounds on what a kernel of 16-bit operands and fp32 sums may be off.

The bounds count roundings (u = eps / 2 of the type, u32 = 2^-24) and nothing else:
  scores    fp32 sums of D exact products, scaled and exponentiated: a weight's relative error is at most
            e_w = 2 ((D + 8) u32 scale max_j sum_d |q_d k_jd| + 2.1e-4 + L 2^-24), twice since the sum of L weights has it
            too; 2.1e-4 covers the softmax's exponentials (each off by at most 1.05e-4).
  O         sum_j P_j v_j with P rounded to 16 bits:  |dO| <= u |O| + (u_p + e_w) sum_j P_j |v_j| + tiny_p sum_j |v_j|
            (over an e4m3 cache the rounded weights are P_j times the values' scales, in fp16: see paged64)
  dV, dK, dQ: see gradients64."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
EXP = 2.1e-4


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Largest absolute error of rounding a value below the type's normal range."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2 if dtype != torch.bfloat16 else 0.0


def rotary64(x, positions, inv_freq, interleaved, scale, sign=1.0):
    """The rotation pair by pair; x [tokens, heads, dim]."""
    r = 2 * inv_freq.numel()
    angle = sign * positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = (angle.cos() * scale)[:, None, :], (angle.sin() * scale)[:, None, :]
    y = x.double().clone()
    ia = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    ib = ia + 1 if interleaved else ia + r // 2
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def quantise_rows(x):
    """(codes e4m3, scale fp32): scale = max|x| / 448 per row, codes = e4m3(x / scale), both divisions in fp32 (IEEE)."""
    f = x.float()
    scale = f.abs().amax(-1) / torch.tensor(448.0, device=x.device)
    q = torch.where(scale[..., None] > 0, f / scale[..., None], torch.zeros_like(f))
    return q.to(torch.float8_e4m3fn), scale


def attention64(q, k, v, allowed, scale, dtype, p_dtype=None, p_tiny=None):
    """One head: q [n, d], k, v [l, d] in any type, allowed [n, l]. P is rounded to p_dtype (default: dtype), with an absolute
    error of p_tiny below its normal range. Returns (O, bound, P, lse, e_w) in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.t() * scale).masked_fill(~allowed, -math.inf)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    some = torch.isfinite(lse)[:, None]
    p = torch.where(some & allowed, torch.exp(s - torch.where(some, lse[:, None], torch.zeros_like(lse[:, None]))), 0.0)
    o = p @ v
    u, pt = half_step(dtype), p_dtype or dtype
    mass = (q.abs() @ k.abs().t()).masked_fill(~allowed, 0.0) * scale
    top = mass.amax(-1, keepdim=True) if k.shape[0] else torch.zeros_like(some, dtype=torch.float64)
    e_w = 2 * ((q.shape[1] + 8) * U32 * top + EXP + max(1, k.shape[0]) * U32)
    reach = (allowed.double() @ v.abs())
    bound = u * o.abs() + (half_step(pt) + e_w) * (p @ v.abs()) + (tiny(pt) if p_tiny is None else p_tiny) * reach + tiny(dtype)
    return o, bound, p, lse, e_w


def gradients64(q, k, v, do, allowed, scale, dtype):
    """One head's O and gradients: dict name -> (value, bound). The kernel's dS uses its own rounded O for the row sums
    and rounds P and dS to 16 bits:
      |d dS| <= (u + e) |dS| + P (sum_d |dO_d| |O error| + (D + 2) u32 (|dO| |v| + |dO| |O|)) + tiny, with e = 2 e_w."""
    o, bo, p, lse, e_w = attention64(q, k, v, allowed, scale, dtype)
    q, k, v, do = q.double(), k.double(), v.double(), do.double()
    u, d, e = half_step(dtype), q.shape[1], 2 * e_w
    dp = do @ v.t()
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    d_delta = (do.abs() * bo).sum(-1, keepdim=True) + (d + 2) * U32 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    t = tiny(dtype) * allowed.double()
    e_ds = (u + e) * ds.abs() + p * (d_delta + (d + 2) * U32 * (do.abs() @ v.abs().t())) + t
    n, l = p.shape
    dv = p.t() @ do
    bv = u * dv.abs() + ((u + e + n * U32) * p + t).t() @ do.abs() + tiny(dtype)
    dq, dk = ds @ k * scale, ds.t() @ q * scale
    bq = u * dq.abs() + scale * ((e_ds + l * U32 * ds.abs()) @ k.abs()) + tiny(dtype)
    bk = u * dk.abs() + scale * ((e_ds + n * U32 * ds.abs()).t() @ q.abs()) + tiny(dtype)
    return {"O": (o, bo), "dQ": (dq, bq), "dK": (dk, bk), "dV": (dv, bv)}


def packed64(q, k, v, lens, causal, scale, do=None):
    """Packed sequences with grouped heads: dict name -> (value, bound) of O (and the gradients when do is given). The sum
    over a group's heads is made before the one rounding of dK and dV; the heads' bounds add up."""
    T, H, D = q.shape
    G = H // k.shape[1]
    names = ["O"] + (["dQ", "dK", "dV"] if do is not None else [])
    shape = {"O": q, "dQ": q, "dK": k, "dV": k}
    out = {n: (torch.zeros(shape[n].shape, dtype=torch.float64, device=q.device),
               torch.zeros(shape[n].shape, dtype=torch.float64, device=q.device)) for n in names}
    a = 0
    for n in lens:
        rows = slice(a, a + n)
        allowed = torch.ones(n, n, dtype=torch.bool, device=q.device)
        allowed = allowed.tril() if causal else allowed
        for h in range(H):
            c = h // G
            if do is None:
                got = {"O": attention64(q[rows, h], k[rows, c], v[rows, c], allowed, scale, q.dtype)[:2]}
            else:
                got = gradients64(q[rows, h], k[rows, c], v[rows, c], do[rows, h], allowed, scale, q.dtype)
            for name, (val, bound) in got.items():
                at = h if name in ("O", "dQ") else c
                out[name][0][rows, at] += val
                out[name][1][rows, at] += bound
        a += n
    return out


def paged64(q, k_cache, v_cache, block_table, kv_lens, new, scale, k_scale=None, v_scale=None):
    """(O, bound) of attention over a paged cache; kv_lens and new are lists. Codes are multiplied by their scales in 64
    bits. With e4m3 codes the weights P_j s_j (s_j: the value's scale; their product is one more fp32 rounding, which e_w's
    factor of two has room for) are rounded to fp16 and meet the codes. They are brought near 1 first, so fp16's absolute
    error of 2^-25 counts in units of the row's largest P_j s_j, or, where the reference is the largest scale alone, of 2^-6
    of that (weights up to 2^7 are left room for): 2^-25 max(max_j P_j s_j, 2^-6 max_j s_j) sum_j |code_j|."""
    T, H, D = q.shape
    kv_heads, page = k_cache.shape[2], k_cache.shape[1]
    G = H // kv_heads
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    b = torch.zeros_like(o)
    a = 0
    for i, (n, L) in enumerate(zip(new, kv_lens)):
        pages = block_table[i, : -(-L // page)].long()

        def rows(cache):
            return torch.stack([cache[p].to(torch.float64) for p in pages.tolist()]).flatten(0, 1)[:L] if L else \
                torch.zeros(0, kv_heads, D, dtype=torch.float64, device=q.device)

        def scales(sc):
            return sc[pages].flatten(0, 1)[:L, :, None].double()

        k, v = rows(k_cache), rows(v_cache)
        if k_scale is not None:
            codes, sv = v.abs(), scales(v_scale)
            k, v = k * scales(k_scale), v * sv
        pos = L - n + torch.arange(n, device=q.device)
        allowed = torch.arange(L, device=q.device)[None, :] <= pos[:, None]
        for h in range(H):
            c = h // G
            if k_scale is None:
                val, bound = attention64(q[a:a + n, h], k[:, c], v[:, c], allowed, scale, q.dtype)[:2]
            else:
                val, bound, p = attention64(q[a:a + n, h], k[:, c], v[:, c], allowed, scale, q.dtype, torch.float16, 0.0)[:3]
                if L:
                    s = sv[:, c, 0]
                    unit = torch.maximum((p * s).amax(-1), (allowed * s).amax(-1) * 2.0 ** -6)
                    bound = bound + tiny(torch.float16) * unit[:, None] * (allowed.double() @ codes[:, c])
            o[a:a + n, h], b[a:a + n, h] = val, bound
        a += n
    return o, b


def worst(got, want, bound) -> float:
    """Largest |got - want| / bound (must be <= 1); any NaN is infinite."""
    r = (got.double() - want).abs() / bound.clamp(min=1e-300)
    r = torch.where((got.double() == want), torch.zeros_like(r), r)
    return float("inf") if torch.isnan(r).any() else float(r.max()) if r.numel() else 0.0
