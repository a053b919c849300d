"""Workloads of the serving and training attention chain: rotary positions, the paged key/value cache (written, also
quantised to e4m3, and read back), attention of new tokens over that cache, and attention over packed prompts.

Every case runs in a plain form (elementary torch operations, fp32) and, with ``own`` set, through the public
functions of ``periodicdent42_b200``. Packed tensors are [tokens, heads, head dim]; caches are
[pages, page size, key/value heads, head dim].
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


def listed():
    return [
        # rotary: one new token for each of 64 running sequences, far positions; latency counts
        {"name": "rotary decode", "op": "rotary", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary_dim": 128,
         "interleaved": False, "dtype": "bf16", "longest": 131072, "attn_scale": 1.0, "backward": False},
        # rotary in training: a packed batch, neighbouring pairs of half the head, scaled for a long context, with gradients
        {"name": "rotary train part head", "op": "rotary", "tokens": 16383, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary_dim": 64, "interleaved": True, "dtype": "bf16", "longest": 16384, "attn_scale": 1.2079, "backward": True},
        # the step's new keys and values of 64 running sequences, quantised as they are written
        {"name": "append decode e4m3", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 64, "pages": 512,
         "dtype": "bf16", "cache": "e4m3"},
        # a long prompt's keys and values, quantised as they are written
        {"name": "append prompt e4m3", "op": "append", "tokens": 16383, "kv_heads": 8, "dim": 128, "page": 64, "pages": 512,
         "dtype": "bf16", "cache": "e4m3"},
        # a cached prefix read back for a prompt that reuses it
        {"name": "gather prefix e4m3", "op": "gather", "tokens": 8191, "kv_heads": 8, "dim": 128, "page": 16, "pages": 1024,
         "dtype": "bf16", "cache": "e4m3"},
        # one user, one new token, a short odd context: latency alone
        {"name": "paged decode single", "op": "paged", "new": "1", "kv": "517", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "cache": "bf16"},
        # a full decode batch over contexts of many lengths, quantised cache
        {"name": "paged decode batch e4m3", "op": "paged", "new": ",".join(["1"] * 64),
         "kv": ",".join(str(97 + 8095 * ((37 * i) % 64) // 63) for i in range(64)), "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "cache": "e4m3"},
        # eight drafted tokens of each of 16 sequences checked at once
        {"name": "paged verify drafts", "op": "paged", "new": ",".join(["8"] * 16),
         "kv": ",".join(str(1000 + 199 * i) for i in range(16)), "heads": 16, "kv_heads": 4, "dim": 64, "page": 128,
         "dtype": "fp16", "cache": "fp16"},
        # chunks of long prompts over their cached contexts
        {"name": "paged chunks long", "op": "paged", "new": "2048,512,77", "kv": "16384,5003,77", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "dtype": "bf16", "cache": "bf16"},
        # a handful of short prompts packed together, forward and gradients, as many key/value heads as query heads
        {"name": "varlen train short", "op": "varlen", "lens": "1,200,37,128,96,255,64,129,3,77", "heads": 8, "kv_heads": 8,
         "dim": 128, "causal": True, "dtype": "bf16", "backward": True},
        # a training batch of packed documents with shared key/value heads, forward and gradients
        {"name": "varlen train packed", "op": "varlen", "lens": "2048,1531,1024,777,2048,515,249", "heads": 16, "kv_heads": 4,
         "dim": 64, "causal": True, "dtype": "fp16", "backward": True},
        # one whole long prompt, forward
        {"name": "varlen prompt 8192", "op": "varlen", "lens": "8192", "heads": 32, "kv_heads": 8, "dim": 128, "causal": True,
         "dtype": "bf16", "backward": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def _list(text):
    return [int(v) for v in text.split(",")]


def draw(rng):
    op = rng.choice(["rotary", "append", "gather", "paged", "paged", "varlen", "varlen"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rotary":
        rotary_dim = rng.choice([dim, dim // 2, dim // 4])
        return {"op": op, "tokens": _log(rng, 1, 16384), "heads": min(heads, 32), "kv_heads": kv_heads, "dim": dim,
                "rotary_dim": rotary_dim, "interleaved": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "longest": _log(rng, 20000, 1000000), "attn_scale": rng.choice([1.0, 1.1386]), "backward": rng.random() < 0.4}
    if op in ("append", "gather"):
        page = rng.choice([16, 32, 64, 128])
        tokens = _log(rng, 1, 16384)
        return {"op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page,
                "pages": -(-tokens // page) + rng.randint(1, 64), "dtype": dtype, "cache": rng.choice([dtype, "e4m3", "e4m3"])}
    if op == "paged":
        batch = _log(rng, 1, 48)
        longest = _log(rng, 64, 12000 if batch < 8 else 4000)
        most = rng.choice([1, 1, 4, _log(rng, 2, 1024)])
        most = min(most, max(1, 4000 // batch), longest)
        new = [rng.randint((most + 1) // 2, most) for _ in range(batch)]
        kv = [n + _log(rng, 1, max(1, longest)) - 1 for n in new]
        return {"op": op, "new": _text(new), "kv": _text(kv), "heads": min(heads, 32), "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "cache": rng.choice([dtype, "e4m3"])}
    backward = rng.random() < 0.6
    longest = _log(rng, 16, 3000 if backward else 5000)
    batch = rng.randint(1, max(1, min(24, 8000 // longest)))
    lens = [max(1, int(longest * rng.random() ** 0.7)) for _ in range(batch - 1)] + [longest]
    return {"op": op, "lens": _text(lens), "heads": min(heads, 24 if backward else 32), "kv_heads": kv_heads, "dim": dim,
            "causal": rng.random() < 0.8, "dtype": dtype, "backward": backward}


def _quantise(x):
    """One scale for each token and head: amax / 448; codes are x / scale in e4m3. A row of zeros has scale 0 and codes 0."""
    x = x.float()
    scale = x.abs().amax(-1) / torch.full((), E4M3_MAX, device=x.device)
    codes = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x)).to(E4M3)
    return codes, scale


def _cu(lens):
    return torch.tensor([0] + lens, device=DEVICE).cumsum(0).to(torch.int32)


def _caches(case, pages, rand, dtype):
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    k, v = rand(shape), rand(shape)
    if case["cache"] != "e4m3":
        return {"k_cache": k.to(dtype), "v_cache": v.to(dtype), "k_scale": None, "v_scale": None}
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    return {"k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def rand(shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    dim = case["dim"]
    if case["op"] == "rotary":
        T = case["tokens"]
        s["q"], s["k"] = rand((T, case["heads"], dim)).to(dtype), rand((T, case["kv_heads"], dim)).to(dtype)
        s["positions"] = torch.randint(0, case["longest"], (T,), generator=g, device=DEVICE)
        half = torch.arange(0, case["rotary_dim"], 2, device=DEVICE, dtype=torch.float64) / case["rotary_dim"]
        s["inv_freq"] = (500000.0 ** -half).float()
        if case["backward"]:
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
            s["dq"], s["dk"] = rand(s["q"].shape).to(dtype), rand(s["k"].shape).to(dtype)
        return s
    if case["op"] in ("append", "gather"):
        T = case["tokens"]
        s.update(_caches(case, case["pages"], rand, dtype))
        s["slots"] = torch.randperm(case["pages"] * case["page"], generator=g, device=DEVICE)[:T]
        if case["op"] == "append":
            s["k"], s["v"] = rand((T, case["kv_heads"], dim)).to(dtype), rand((T, case["kv_heads"], dim)).to(dtype)
        return s
    if case["op"] == "paged":
        new, kv = _list(case["new"]), _list(case["kv"])
        width = -(-max(kv) // case["page"])
        need = [-(-n // case["page"]) for n in kv]
        pages = sum(need) + 3
        s.update(_caches(case, pages, rand, dtype))
        order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        first = torch.tensor([0] + need[:-1], device=DEVICE).cumsum(0)
        at = first[:, None] + torch.arange(width, device=DEVICE)
        used = torch.arange(width, device=DEVICE) < torch.tensor(need, device=DEVICE)[:, None]
        s["block_table"] = torch.where(used, order[at.clamp(max=pages - 1)], torch.zeros_like(order[:1])).contiguous()
        s["kv_lens"] = torch.tensor(kv, device=DEVICE, dtype=torch.int32)
        s["cu_seqlens"] = _cu(new)
        s["most_new"], s["most_kv"] = max(new), max(kv)
        s["q"] = rand((sum(new), case["heads"], dim)).to(dtype)
        return s
    lens = _list(case["lens"])
    T = sum(lens)
    s["cu_seqlens"], s["most"] = _cu(lens), max(lens)
    s["q"] = rand((T, case["heads"], dim)).to(dtype)
    s["k"], s["v"] = rand((T, case["kv_heads"], dim)).to(dtype), rand((T, case["kv_heads"], dim)).to(dtype)
    if case["backward"]:
        for n in "qkv":
            s[n].requires_grad_(True)
        s["do"] = rand((T, case["heads"], dim)).to(dtype)
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, positions, inv_freq, interleaved, scale):
    """Angles in 64 bits (far positions), the rotation in 32."""
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * scale).float()[:, None]
    r = 2 * inv_freq.numel()
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2 : r])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _padded(x, cu, most):
    """[batch, most, ...] rows of the packed x and which of them exist; the others are zero."""
    at = cu[:-1, None].long() + torch.arange(most, device=x.device)
    real = at < cu[1:, None]
    rows = x[at.clamp(max=x.shape[0] - 1)].float()
    return torch.where(real[:, :, None, None], rows, torch.zeros((), device=x.device)), real


def _packed(x, real):
    return x[real]


def _attend(q, k, v, mask, scale):
    """q [b, n, heads, d], k and v [b, l, kv heads, d], mask [b, n, l]; rows without keys give zero."""
    b, n, h, d = q.shape
    g = k.shape[2]
    qs = q.view(b, n, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(b, g, (h // g) * n, d)
    s = torch.matmul(qs, k.permute(0, 2, 3, 1)) * scale
    s = s.view(b, g, h // g, n, -1).masked_fill(~mask[:, None, None], -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, g, (h // g) * n, -1), v.transpose(1, 2)).view(b, g, h // g, n, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d)


def _rows(cache, scale, at):
    """The cached rows `at` in 32 bits: codes times their scale where the cache is quantised."""
    flat = cache.view(-1, *cache.shape[2:])
    if scale is None:
        return flat[at].float()
    return flat.view(torch.uint8)[at].view(E4M3).float() * scale.view(-1, scale.shape[-1])[at][..., None]


def _plain_paged(s):
    q, real = _padded(s["q"], s["cu_seqlens"], s["most_new"])
    here = torch.arange(s["most_kv"], device=DEVICE)
    lens = s["kv_lens"].long()
    at = s["block_table"].long()[:, here // s["page"]] * s["page"] + here % s["page"]
    held = (here < lens[:, None])[:, :, None, None]
    k = torch.where(held, _rows(s["k_cache"], s["k_scale"], at), torch.zeros((), device=DEVICE))
    v = torch.where(held, _rows(s["v_cache"], s["v_scale"], at), torch.zeros((), device=DEVICE))
    place = (lens - (s["cu_seqlens"][1:] - s["cu_seqlens"][:-1]))[:, None] + torch.arange(s["most_new"], device=DEVICE)
    mask = (here <= place[:, :, None]) & (here < lens[:, None])[:, None]
    return _packed(_attend(q, k, v, mask, s["dim"] ** -0.5), real).to(s["q"].dtype)


def _plain_varlen(s):
    cu, most = s["cu_seqlens"], s["most"]
    (q, real), (k, _), (v, _) = (_padded(s[n], cu, most) for n in "qkv")
    here = torch.arange(most, device=DEVICE)
    mask = real[:, None, :].expand(-1, most, -1)
    if s["causal"]:
        mask = mask & (here[None, :] <= here[:, None])
    return _packed(_attend(q, k, v, mask, s["dim"] ** -0.5), real).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        import periodicdent42_b200 as bsk
    op = s["op"]
    if op == "rotary":
        if own:
            q, k = bsk.rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"],
                                        scale=s["attn_scale"])
        else:
            q, k = (_rotate(s[n], s["positions"], s["inv_freq"], s["interleaved"], s["attn_scale"]) for n in "qk")
        if not s["backward"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return q.detach(), k.detach(), dq, dk
    if op == "append":
        if own:
            bsk.kv_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        elif s["k_scale"] is None:
            s["k_cache"].view(-1, s["kv_heads"], s["dim"])[s["slots"]] = s["k"]
            s["v_cache"].view(-1, s["kv_heads"], s["dim"])[s["slots"]] = s["v"]
        else:
            (kc, ks), (vc, vs) = _quantise(s["k"]), _quantise(s["v"])
            s["k_cache"].view(torch.uint8).view(-1, s["kv_heads"], s["dim"])[s["slots"]] = kc.view(torch.uint8)
            s["v_cache"].view(torch.uint8).view(-1, s["kv_heads"], s["dim"])[s["slots"]] = vc.view(torch.uint8)
            s["k_scale"].view(-1, s["kv_heads"])[s["slots"]] = ks
            s["v_scale"].view(-1, s["kv_heads"])[s["slots"]] = vs
        return [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None]
    if op == "gather":
        dtype = DTYPES[s["dtype"]]
        if own:
            return bsk.kv_cache_gather(s["k_cache"], s["v_cache"], s["slots"], dtype=dtype, k_scale=s["k_scale"], v_scale=s["v_scale"])
        return _rows(s["k_cache"], s["k_scale"], s["slots"]).to(dtype), _rows(s["v_cache"], s["v_scale"], s["slots"]).to(dtype)
    if op == "paged":
        if own:
            return bsk.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["cu_seqlens"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"])
        return _plain_paged(s)
    if own:
        o = bsk.attention_varlen(s["q"], s["k"], s["v"], s["cu_seqlens"], causal=s["causal"])
    else:
        o = _plain_varlen(s)
    if not s["backward"]:
        return o
    return o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def work(case):
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    h, g, d = case.get("heads", 0), case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        T, ways = case["tokens"], 2 if case["backward"] else 1
        return {"bytes": ways * 2 * T * (h + g) * d * e + 8 * T, "flops": ways * 3 * T * (h + g) * case["rotary_dim"]}
    if case["op"] in ("append", "gather"):
        T, held = case["tokens"], (1 + 4 / d) if case["cache"] == "e4m3" else e
        return {"bytes": int(2 * T * g * d * (e + held)) + 8 * T, "flops": 2 * T * g * d * (2 if case["cache"] == "e4m3" else 0)}
    if case["op"] == "paged":
        new, kv = _list(case["new"]), _list(case["kv"])
        held = (1 + 4 / d) if case["cache"] == "e4m3" else e
        pairs = sum(sum(max(0, L - n + t + 1) for t in range(n)) for n, L in zip(new, kv))
        return {"bytes": int(2 * sum(kv) * g * d * held + 2 * sum(new) * h * d * e), "flops": 4 * pairs * h * d}
    lens = _list(case["lens"])
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
    T = sum(lens)
    once = T * (2 * h + 2 * g) * d * e
    if not case["backward"]:
        return {"bytes": once, "flops": 4 * pairs * h * d}
    # the gradients read q, k, v, o and do and write dq, dk and dv; five products, one of them the scores again
    return {"bytes": once + T * (4 * h + 4 * g) * d * e, "flops": 14 * pairs * h * d}


# ------------------------------------------------------------------------------------------------- 64 bits
def _turn64(x, s, sign):
    """The rotation as a complex product of each pair with scale * e^(i * sign * angle)."""
    r = s["rotary_dim"]
    angle = sign * torch.outer(s["positions"].double(), s["inv_freq"].double())
    unit = torch.polar(torch.full_like(angle, s["attn_scale"]), angle)[:, None]
    y = x.detach().double().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if s["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _softmax64(q, k, allowed):
    p = torch.softmax((q @ k.t() / math.sqrt(q.shape[1])).masked_fill(~allowed, -math.inf), -1)
    return torch.nan_to_num(p)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        out = [_turn64(s["q"], s, 1), _turn64(s["k"], s, 1)]
        if case["backward"]:
            out += [_turn64(s["dq"], s, -1), _turn64(s["dk"], s, -1)]
        return tuple(out)
    if op == "append":
        page, off = s["slots"] // case["page"], s["slots"] % case["page"]
        caches, scales = [], []
        for n in "kv":
            x = s[n].double()
            if s[n + "_scale"] is None:
                caches.append(s[n + "_cache"].double().index_put((page, off), x))
            else:  # the codes are 8-bit values without a counterpart in 64 bits
                caches.append(None)
                scales.append(s[n + "_scale"].double().index_put((page, off), x.abs().amax(-1) / 448))
        return caches + scales
    if op == "gather":
        out = []
        for n in "kv":
            page, off = s["slots"] // case["page"], s["slots"] % case["page"]
            x = s[n + "_cache"].double()[page, off]
            out.append(x if s[n + "_scale"] is None else x * s[n + "_scale"].double()[page, off].unsqueeze(-1))
        return tuple(out)
    h, g = case["heads"], case["kv_heads"]
    q = s["q"].detach().double()
    o = torch.zeros_like(q)
    if op == "paged":
        first = 0
        for i, (n, L) in enumerate(zip(_list(case["new"]), _list(case["kv"]))):
            pages = s["block_table"][i, : -(-L // case["page"])].long()
            kv = {}
            for m in "kv":
                kv[m] = s[m + "_cache"].view(torch.uint8)[pages].view(s[m + "_cache"].dtype).double()
                if s[m + "_scale"] is not None:
                    kv[m] = kv[m] * s[m + "_scale"][pages].double()[..., None]
                kv[m] = kv[m].flatten(0, 1)[:L]
            allowed = torch.ones(n, L, dtype=torch.bool, device=DEVICE).tril(L - n)
            for a in range(h):
                c = a * g // h
                o[first : first + n, a] = _softmax64(q[first : first + n, a], kv["k"][:, c], allowed) @ kv["v"][:, c]
            first += n
        return o
    k, v = s["k"].detach().double(), s["v"].detach().double()
    back = case["backward"]
    if back:
        do = s["do"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    first = 0
    for n in _list(case["lens"]):
        at = slice(first, first + n)
        allowed = torch.ones(n, n, dtype=torch.bool, device=DEVICE)
        allowed = allowed.tril() if case["causal"] else allowed
        for a in range(h):
            c = a * g // h
            p = _softmax64(q[at, a], k[at, c], allowed)
            o[at, a] = p @ v[at, c]
            if back:
                dv[at, c] += p.t() @ do[at, a]
                ds = p * (do[at, a] @ v[at, c].t() - (do[at, a] * o[at, a]).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
                dq[at, a] = ds @ k[at, c]
                dk[at, c] += ds.t() @ q[at, a]
        first += n
    return (o, dq, dk, dv) if back else o
