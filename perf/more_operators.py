"""Workloads of a decoder layer with a sliding attention window: attention of packed sequences (with gradients) and of new
tokens over a paged cache where a token sees a window of the last keys and a few first ones; norms of each head of the
queries and keys with the rotation in the same pass; rotary positions with several axes; and a serving step's block tables,
slots and positions from the requests' lengths.

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
EPS = 1e-6


def listed():
    return [
        # one user, one new token, a window over an odd context: latency alone
        {"name": "window decode single", "op": "paged", "new": "1", "kv": "1301", "window": 512, "sinks": 4, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "cache": "bf16"},
        # a full decode batch over long contexts of many lengths, quantised cache
        {"name": "window decode batch e4m3", "op": "paged", "new": ",".join(["1"] * 64),
         "kv": ",".join(str(97 + 16287 * ((37 * i) % 64) // 63) for i in range(64)), "window": 1024, "sinks": 4, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "cache": "e4m3"},
        # chunks of long prompts over their cached contexts
        {"name": "window chunks", "op": "paged", "new": "2048,512,77", "kv": "16384,5003,77", "window": 1024, "sinks": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "dtype": "bf16", "cache": "bf16"},
        # a handful of short documents packed together, forward and gradients, as many key/value heads as query heads
        {"name": "window train short", "op": "varlen", "lens": "1,200,37,128,96,255,64,129,3,77", "window": 64, "sinks": 1,
         "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "fp16", "backward": True},
        # a training batch of packed long documents with shared key/value heads, forward and gradients
        {"name": "window train packed", "op": "varlen", "lens": "8192,4096,2500,1000,596", "window": 1024, "sinks": 4,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "backward": True},
        # one whole long prompt, forward
        {"name": "window prompt 32768", "op": "varlen", "lens": "32768", "window": 4096, "sinks": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "backward": False},
        # the step's new queries and keys of 64 running sequences, far positions; latency counts
        {"name": "norm rotary decode", "op": "norm", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary_dim": 128,
         "interleaved": False, "sections": "", "cycle": False, "dtype": "bf16", "weights": "bf16", "longest": 131072,
         "attn_scale": 1.0, "backward": False},
        # a training batch, with the gradients of queries, keys and both weights
        {"name": "norm rotary train", "op": "norm", "tokens": 16383, "heads": 32, "kv_heads": 8, "dim": 128, "rotary_dim": 128,
         "interleaved": False, "sections": "", "cycle": False, "dtype": "bf16", "weights": "fp32", "longest": 16384,
         "attn_scale": 1.0, "backward": True},
        # one small image's patches in an encoder: rows and columns
        {"name": "axes image", "op": "axes", "tokens": 257, "heads": 16, "kv_heads": 16, "dim": 64, "rotary_dim": 64,
         "interleaved": False, "sections": "16,16", "cycle": False, "dtype": "bf16", "longest": 64, "attn_scale": 1.0,
         "backward": False},
        # text, images and video packed for training: time, rows and columns in turn, with gradients
        {"name": "axes video train", "op": "axes", "tokens": 16383, "heads": 32, "kv_heads": 8, "dim": 128, "rotary_dim": 128,
         "interleaved": False, "sections": "24,20,20", "cycle": True, "dtype": "bf16", "longest": 16384, "attn_scale": 1.0,
         "backward": True},
        # one decode step of 64 running requests: most tokens land in a page that is there, some open one
        {"name": "plan decode", "op": "plan", "new": ",".join(["1"] * 64),
         "kv": ",".join(str(97 + 8095 * ((37 * i) % 64) // 63) for i in range(64)), "page": 64, "padding": 0, "spare": 100},
        # prompts of many lengths admitted beside running requests, rows padded for a captured graph
        {"name": "plan prompts", "op": "plan", "new": ",".join(str(1 if i % 3 else 1 + (i * 7919) % 499) for i in range(200)),
         "kv": ",".join(str((i * 911) % 3001 if i % 3 else 0) for i in range(200)), "page": 16, "padding": 517, "spare": 33},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def _list(text):
    return [int(v) for v in text.split(",")]


def draw(rng):
    op = rng.choice(["paged", "paged", "varlen", "varlen", "norm", "axes", "plan"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = min(kv_heads * rng.choice([1, 2, 3, 4, 5, 8]), 32)
    heads -= heads % kv_heads
    dtype = rng.choice(["bf16", "fp16"])
    if op == "plan":
        batch = _log(rng, 1, 400)
        longest = _log(rng, 1, max(1, 16000 // batch))
        new = [rng.choice([1, rng.randint(0, longest)]) for _ in range(batch)]
        return {"op": op, "new": _text(new), "kv": _text([rng.choice([0, _log(rng, 1, 8000)]) for _ in range(batch)]),
                "page": rng.choice([8, 16, 32, 64, 128]), "padding": rng.choice([0, rng.randint(1, 600)]),
                "spare": rng.randint(0, 200)}
    if op in ("norm", "axes"):
        dim = rng.choice([64, 80, 96, 128, 256])
        rotary_dim = rng.choice([dim, dim, dim // 2])
        parts = rng.choice([2, 3]) if op == "axes" or rng.random() < 0.3 else 0
        sections = ""
        if parts:
            pairs = rotary_dim // 2
            cut = sorted(rng.randint(0, pairs) for _ in range(parts - 1))
            sections = _text([b - a for a, b in zip([0] + cut, cut + [pairs])])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        case = {"op": op, "tokens": _log(rng, 1, 16384 * 128 // max(dim, 128)), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary_dim": rotary_dim, "interleaved": rng.random() < 0.5, "sections": sections, "cycle": rng.random() < 0.5,
                "dtype": dtype, "longest": _log(rng, 20, 1000000), "attn_scale": rng.choice([1.0, 1.1386]),
                "backward": rng.random() < 0.5}
        if op == "norm":
            case["weights"] = rng.choice([dtype, "fp32"])
        return case
    window = _log(rng, 1, 4096)
    sinks = rng.choice([0, 0, 1, 4, _log(rng, 2, 300)])
    if op == "paged":
        batch = _log(rng, 1, 48)
        longest = _log(rng, 64, 24000 if batch < 8 else 6000)
        most = rng.choice([1, 1, 4, _log(rng, 2, 1024)])
        most = min(most, max(1, 4000 // batch), longest)
        new = [rng.randint((most + 1) // 2, most) for _ in range(batch)]
        kv = [n + _log(rng, 1, longest) - 1 for n in new]
        return {"op": op, "new": _text(new), "kv": _text(kv), "window": window, "sinks": sinks, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "dtype": dtype,
                "cache": rng.choice([dtype, "e4m3"])}
    backward = rng.random() < 0.6
    longest = _log(rng, 16, 12000)
    batch = rng.randint(1, max(1, min(24, 12000 // longest)))
    lens = [max(1, int(longest * rng.random() ** 0.7)) for _ in range(batch - 1)] + [longest]
    return {"op": op, "lens": _text(lens), "window": window, "sinks": sinks, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "backward": backward}


def _quantise(x):
    """One scale for each token and head: amax / 448; codes are x / scale in e4m3."""
    x = x.float()
    scale = x.abs().amax(-1) / E4M3_MAX
    codes = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x)).to(E4M3)
    return codes, scale


def _cu(lens):
    return torch.tensor([0] + lens, device=DEVICE).cumsum(0).to(torch.int32)


def _axis_list(case):
    """Which axis each pair takes: runs of the sections, or the axes in turn, passing over those whose section is used up."""
    left = _list(case["sections"])
    if not case["cycle"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def rand(shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = dict(case)
    if case["op"] == "plan":
        new, kv = _list(case["new"]), _list(case["kv"])
        page = case["page"]
        have, need = [-(-k // page) for k in kv], [-(-(k + n) // page) for k, n in zip(kv, new)]
        width = max(max(need), 1) + 2
        pages = sum(need) + case["spare"]
        order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
        # the requests' pages are the first of the order, the free ones the rest; behind the free ones the stack holds old entries
        at = torch.tensor([0] + have[:-1], device=DEVICE).cumsum(0)[:, None] + torch.arange(width, device=DEVICE)
        held = torch.arange(width, device=DEVICE) < torch.tensor(have, device=DEVICE)[:, None]
        s["block_table"] = torch.where(held, order[at.clamp(max=pages - 1)], torch.full_like(order[:1], -1)).contiguous()
        s["free_pages"] = torch.cat([order[sum(have):], order[: sum(have)]]).contiguous()
        s["free_count"] = torch.tensor([pages - sum(have)], device=DEVICE, dtype=torch.int32)
        s["kv_lens"] = torch.tensor(kv, device=DEVICE, dtype=torch.int32)
        s["new_lens"] = torch.tensor(new, device=DEVICE, dtype=torch.int32)
        s["tokens"] = sum(new) + case["padding"]
        return s
    dtype = DTYPES[case["dtype"]]
    dim = case["dim"]
    if case["op"] in ("norm", "axes"):
        T = case["tokens"]
        s["q"], s["k"] = rand((T, case["heads"], dim)).to(dtype), rand((T, case["kv_heads"], dim)).to(dtype)
        half = torch.arange(0, case["rotary_dim"], 2, device=DEVICE, dtype=torch.float64) / case["rotary_dim"]
        s["inv_freq"] = (500000.0 ** -half).float()
        s["axes"] = None
        shape = (T,)
        if case["sections"]:
            shape = (len(_list(case["sections"])), T)
            s["axes"] = torch.tensor(_axis_list(case), device=DEVICE, dtype=torch.int32)
        s["positions"] = torch.randint(0, case["longest"], shape, generator=g, device=DEVICE)
        leaves = ["q", "k"]
        if case["op"] == "norm":
            for n in "qk":
                s["w" + n] = (1.0 + 0.2 * rand((dim,))).to(DTYPES[case["weights"]])
            leaves += ["wq", "wk"]
        s["leaves"] = leaves
        if case["backward"]:
            for n in leaves:
                s[n].requires_grad_(True)
            s["dq"], s["dk"] = rand(s["q"].shape).to(dtype), rand(s["k"].shape).to(dtype)
        return s
    if case["op"] == "paged":
        new, kv = _list(case["new"]), _list(case["kv"])
        width = -(-max(kv) // case["page"])
        need = [-(-n // case["page"]) for n in kv]
        pages = sum(need) + 3
        shape = (pages, case["page"], case["kv_heads"], dim)
        for n in "kv":
            x = rand(shape)
            s[n + "_cache"], s[n + "_scale"] = _quantise(x) if case["cache"] == "e4m3" else (x.to(dtype), None)
            del x
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
def _rotate(y, s):
    """Angles in 64 bits (far positions), the rotation in 32; y in 32 bits."""
    at = s["positions"][s["axes"].long()].t() if s["axes"] is not None else s["positions"][:, None]
    angle = at.double() * s["inv_freq"].double()
    cos, sin = (angle.cos() * s["attn_scale"]).float()[:, None], (angle.sin() * s["attn_scale"]).float()[:, None]
    r = s["rotary_dim"]
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if s["interleaved"] else (y[..., : r // 2], y[..., r // 2 : r])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if s["interleaved"] else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., r:]), -1)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _attend(q, place, lens, keys, values, window, sinks, scale):
    """q [b, n, heads, d] in 32 bits; row t of sequence i stands at place[i, t] and sees the keys j <= place that are among the
    last `window` or the first `sinks`. keys(at), values(at): rows [b, l, kv heads, d] at positions at [b, l]. Rows without
    keys give zero. 512 rows at a time, over the keys that they can see."""
    b, n, h, d = q.shape
    outs = []
    for c0 in range(0, n, 512):
        c = min(512, n - c0)
        near = place[:, c0, None] - window + 1 + torch.arange(window + c - 1, device=q.device)
        far = torch.arange(sinks, device=q.device).expand(b, sinks)
        at = torch.cat((far, near), 1)
        held = (at >= 0) & (at < lens[:, None]) & ((at >= sinks) | (torch.arange(at.shape[1], device=q.device) < sinks))
        here = place[:, c0 : c0 + c, None]
        mask = held[:, None] & (at[:, None] <= here) & ((at[:, None] > here - window) | (at[:, None] < sinks))
        at = torch.where(held, at, torch.zeros_like(at))
        zero = torch.zeros((), device=q.device)
        k, v = (torch.where(held[:, :, None, None], f(at), zero) for f in (keys, values))
        g = k.shape[2]
        qs = q[:, c0 : c0 + c].reshape(b, c, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(b, g, (h // g) * c, d)
        s = torch.matmul(qs, k.permute(0, 2, 3, 1)) * scale
        s = s.view(b, g, h // g, c, -1).masked_fill(~mask[:, None, None], -math.inf)
        top = s.detach().amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, zero, top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(b, g, (h // g) * c, -1), v.transpose(1, 2)).view(b, g, h // g, c, d)
        o = o / torch.where(total > 0, total, torch.ones_like(total))
        outs.append(o.permute(0, 3, 1, 2, 4).reshape(b, c, h, d))
    return torch.cat(outs, 1)


def _rows_of(cu, most, x):
    """[batch, most, ...] rows of the packed x in 32 bits and which of them exist."""
    at = cu[:-1, None].long() + torch.arange(most, device=x.device)
    real = at < cu[1:, None]
    return x[at.clamp(max=x.shape[0] - 1)].float(), real


def _plain_paged(s):
    q, real = _rows_of(s["cu_seqlens"], s["most_new"], s["q"])
    lens = s["kv_lens"].long()
    new = (s["cu_seqlens"][1:] - s["cu_seqlens"][:-1]).long()
    place = (lens - new)[:, None] + torch.arange(s["most_new"], device=DEVICE)

    def rows(n):
        cache, scale = s[n + "_cache"], s[n + "_scale"]
        flat = cache.view(-1, *cache.shape[2:])

        def of(at):
            slot = s["block_table"].long().gather(1, at // s["page"]) * s["page"] + at % s["page"]
            if scale is None:
                return flat[slot].float()
            return flat.view(torch.uint8)[slot].view(E4M3).float() * scale.view(-1, scale.shape[-1])[slot][..., None]

        return of

    window = min(s["window"], s["most_kv"])
    return _attend(q, place, lens, rows("k"), rows("v"), window, s["sinks"], s["dim"] ** -0.5)[real].to(s["q"].dtype)


def _plain_varlen(s):
    cu, most = s["cu_seqlens"].long(), s["most"]
    q, real = _rows_of(cu, most, s["q"])
    place = torch.arange(most, device=DEVICE).expand(cu.shape[0] - 1, most)
    k, v = s["k"].float(), s["v"].float()

    def rows(x):
        return lambda at: x[(cu[:-1, None] + at).clamp(max=x.shape[0] - 1)]

    o = _attend(q, place, cu[1:] - cu[:-1], rows(k), rows(v), min(s["window"], most), s["sinks"], s["dim"] ** -0.5)
    return o[real].to(s["q"].dtype)


def _plain_plan(s):
    page, kv, new, table = s["page"], s["kv_lens"].long(), s["new_lens"].long(), s["block_table"]
    cu = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0)))
    have, need = (kv + page - 1) // page, (kv + new + page - 1) // page
    add = need - have
    first = add.cumsum(0) - add  # pages taken by the requests before
    top = s["free_count"].long() - 1
    cell = torch.arange(table.shape[1], device=DEVICE)
    take = (top - (first[:, None] + cell - have[:, None])).clamp(0, s["free_pages"].shape[0] - 1)
    opened = (cell >= have[:, None]) & (cell < need[:, None])
    table.copy_(torch.where(opened, s["free_pages"][take], table))
    row = torch.arange(s["tokens"], device=DEVICE)
    real = row < cu[-1]
    i = torch.searchsorted(cu[1:], row, right=True).clamp(max=kv.shape[0] - 1)
    at = kv[i] + row - cu[i]
    cell = (at // page).clamp(0, table.shape[1] - 1)
    slots = table[i, cell].long() * page + at % page
    slots, at = torch.where(real, slots, torch.full_like(slots, -1)), torch.where(real, at, torch.zeros_like(at))
    return slots, at.int(), cu.int(), (kv + new).int(), (s["free_count"] - add.sum()).int()


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        import periodicdent42_b200 as bsk
    op = s["op"]
    if op == "plan":
        if own:
            out = bsk.kv_cache_plan(s["kv_lens"], s["new_lens"], s["block_table"], s["free_pages"], s["free_count"], s["page"],
                                    s["tokens"])
        else:
            out = _plain_plan(s)
        return *out, s["block_table"]
    if op in ("norm", "axes"):
        if own and op == "norm":
            q, k = bsk.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["inv_freq"],
                                      interleaved=s["interleaved"], scale=s["attn_scale"], eps=EPS, axes=s["axes"])
        elif own:
            q, k = bsk.rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"],
                                        scale=s["attn_scale"], axes=s["axes"])
        elif op == "norm":
            q, k = (_rotate(_normed(s[n].float(), s["w" + n].float()), s).to(s[n].dtype) for n in "qk")
        else:
            q, k = (_rotate(s[n].float(), s).to(s[n].dtype) for n in "qk")
        if not s["backward"]:
            return q, k
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), [s[n] for n in s["leaves"]], (s["dq"], s["dk"]))
    if op == "paged":
        if own:
            return bsk.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_lens"], s["cu_seqlens"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"], window=s["window"], sinks=s["sinks"])
        return _plain_paged(s)
    if own:
        o = bsk.attention_varlen(s["q"], s["k"], s["v"], s["cu_seqlens"], window=s["window"], sinks=s["sinks"])
    else:
        o = _plain_varlen(s)
    if not s["backward"]:
        return o
    return o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def _pairs(first, n, window, sinks):
    """Keys seen by rows at positions first .. first + n - 1, summed."""
    return sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(max(first, 0), first + n))


def work(case):
    if case["op"] == "plan":
        new, kv = _list(case["new"]), _list(case["kv"])
        opened = sum(-(-(k + n) // case["page"]) - -(-k // case["page"]) for k, n in zip(kv, new))
        tokens = sum(new) + case["padding"]
        # lengths read and written, offsets, slots and positions, pages taken and entered
        return {"bytes": 16 * len(new) + 12 * tokens + 8 * opened, "flops": 4 * tokens}
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("norm", "axes"):
        T, r = case["tokens"], case["rotary_dim"]
        axes = len(_list(case["sections"])) if case["sections"] else 1
        rows = T * (h + g) * d
        if case["op"] == "axes":
            ways = 2 if case["backward"] else 1
            return {"bytes": ways * 2 * rows * e + 8 * T * axes, "flops": ways * 3 * T * (h + g) * r}
        # forward: x read, y written; gradients: x and dy read, dx written
        return {"bytes": (5 if case["backward"] else 2) * rows * e + 8 * T * axes,
                "flops": 4 * rows + 3 * T * (h + g) * r + (9 * rows + 3 * T * (h + g) * r if case["backward"] else 0)}
    window, sinks = case["window"], case["sinks"]
    if case["op"] == "paged":
        new, kv = _list(case["new"]), _list(case["kv"])
        held = (1 + 4 / d) if case["cache"] == "e4m3" else e
        pairs = sum(_pairs(L - n, n, window, sinks) for n, L in zip(new, kv))
        seen = sum(min(L, window + n - 1) + min(sinks, max(0, L - (window + n - 1))) for n, L in zip(new, kv))
        return {"bytes": int(2 * seen * g * d * held + 2 * sum(new) * h * d * e), "flops": 4 * pairs * h * d}
    lens = _list(case["lens"])
    pairs = sum(_pairs(0, n, window, sinks) for n in lens)
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
    pos = s["positions"].double()
    if s["axes"] is None:
        angle = sign * torch.outer(pos, s["inv_freq"].double())
    else:
        angle = sign * torch.stack([pos[a] * f for a, f in zip(s["axes"].tolist(), s["inv_freq"].double().tolist())], 1)
    unit = torch.polar(torch.full_like(angle, s["attn_scale"]), angle)[:, None]
    y = x.detach().double().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if s["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_norm(s):
    outs, dxs, dws = [], [], []
    for n in "qk":
        x, w = s[n].detach().double(), s["w" + n].detach().double()
        rms = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        unit = x / rms
        outs.append(_turn64(unit * w, s, 1))
        if s["backward"]:
            dz = _turn64(s["d" + n], s, -1)
            dws.append((dz * unit).sum((0, 1)))
            dxs.append((dz * w - unit * (dz * w * unit).mean(-1, keepdim=True)) / rms)
    return tuple(outs + dxs + dws)


def _exact_plan(s):
    """Request by request, with the stack of free pages as a list."""
    page = s["page"]
    table = [row[:] for row in s["block_table"].tolist()]
    stack = s["free_pages"].tolist()[: int(s["free_count"])]
    slots, places, cu, after = [], [], [0], []
    for i, (k, n) in enumerate(zip(s["kv_lens"].tolist(), s["new_lens"].tolist())):
        for p in range(k, k + n):
            if p % page == 0:
                table[i][p // page] = stack.pop()
            slots.append(table[i][p // page] * page + p % page)
            places.append(p)
        cu.append(cu[-1] + n)
        after.append(k + n)
    rest = s["tokens"] - len(slots)

    def ints(x):
        return torch.tensor(x, device=DEVICE, dtype=torch.int64)

    return ints(slots + [-1] * rest), ints(places + [0] * rest), ints(cu), ints(after), ints([len(stack)]), ints(table)


def _head64(q, k, v, allowed):
    p = torch.nan_to_num(torch.softmax((q @ k.t() / math.sqrt(q.shape[1])).masked_fill(~allowed, -math.inf), -1))
    return p, p @ v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return _exact_plan(s)
    if op == "norm":
        return _exact_norm(s)
    if op == "axes":
        out = [_turn64(s["q"], s, 1), _turn64(s["k"], s, 1)]
        if case["backward"]:
            out += [_turn64(s["dq"], s, -1), _turn64(s["dk"], s, -1)]
        return tuple(out)
    h, g = case["heads"], case["kv_heads"]
    window, sinks = case["window"], case["sinks"]
    q = s["q"].detach().double()
    o = torch.zeros_like(q)
    back = case.get("backward", False)
    if op == "paged":
        news, lens = _list(case["new"]), _list(case["kv"])
    else:
        news = lens = _list(case["lens"])
        k_all, v_all = s["k"].detach().double(), s["v"].detach().double()
    if back:
        do = s["do"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k_all), torch.zeros_like(v_all)
    first = 0
    for i, (n, L) in enumerate(zip(news, lens)):
        if op == "paged":
            pages = s["block_table"][i, : -(-L // case["page"])].long()
            kv = []
            for m in "kv":
                x = s[m + "_cache"].view(torch.uint8)[pages].view(s[m + "_cache"].dtype).double()
                if s[m + "_scale"] is not None:
                    x = x * s[m + "_scale"][pages].double()[..., None]
                kv.append(x.flatten(0, 1)[:L])
            k, v = kv
        else:
            k, v = k_all[first : first + n], v_all[first : first + n]
        key = torch.arange(L, device=DEVICE)
        for r0 in range(0, n, 2048):  # a band of rows at a time
            r1 = min(n, r0 + 2048)
            at = (L - n + torch.arange(r0, r1, device=DEVICE))[:, None]
            allowed = (key <= at) & ((at - key < window) | (key < sinks))
            rows = slice(first + r0, first + r1)
            for a in range(h):
                c = a * g // h
                p, o[rows, a] = _head64(q[rows, a], k[:, c], v[:, c], allowed)
                if back:
                    cols = slice(first, first + n)
                    dv[cols, c] += p.t() @ do[rows, a]
                    ds = p * (do[rows, a] @ v[:, c].t() - (do[rows, a] * o[rows, a]).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
                    dq[rows, a] = ds @ k[:, c]
                    dk[cols, c] += ds.t() @ q[rows, a]
        first += n
    return (o, dq, dk, dv) if back else o
