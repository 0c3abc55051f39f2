"""The operators of a key/value cache in pages of 8-bit values, measured through the public entry points: `ext.paged_append`
(the step's keys and values normed, rotated, coded and put into the pages, the queries rotated beside them) and
`ext.paged_attention` (attention of one token up to whole chunks over those pages, plain or with capped scores, a bias that
falls with the distance, a sliding window or a prefix that every token sees).

A case is a dict of plain values:
  op       "append" or "attend"
  rows     sequences; "tokens" the new tokens of a row (of the longest one, with "ragged": then the others have fewer, and with
           "ragged" "mixed" all but the first have one); "context" cached positions before them (the rows hold 3/4 to all of it)
  hq, hkv, hd, rot, page   query heads, key/value heads, head size, rotated dims, tokens per page
  norm     (append) RMS norms of queries and keys before the rotation
  cap, window, slopes, prefix   (attend) the options: 0 and false are off
The lengths follow from the case, everything else from (case, seed) by torch generators on the GPU.

The cache: keys e4m3 [pages][hkv][page][hd], values e4m3 [pages][hkv][page / 16][hd][16], each times a power of two per page and
head, held as an E8M0 byte. Appending gives a page the smallest power of two that its largest value fits (a page begun anew
forgets its old one; a page that goes on keeps its own unless the new tokens need a larger one, and then what it held is
coded again). The cache comes back as its e4m3 values and its scales, the bytes' own types and no other bytes.
"""

import math
import os
import random
import sys
import zlib

import torch

own = False

F32, F64, BF16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float8_e4m3fn
EPS, THETA = 1e-6, 1e7
M27 = dict(hq=24, hkv=4, hd=256, rot=64, page=64)  # the 27B model's attention heads
G128 = dict(hq=32, hkv=8, hd=128, rot=128)  # generic grouped heads, rotated whole
M64 = dict(hq=16, hkv=16, hd=64, rot=64)  # generic: a key/value head for every query head


def _case(name, op, heads, rows, tokens, context, ragged="", norm=False, cap=0.0, window=0, slopes=False, prefix=0, **more):
    return {"name": name, "op": op, "rows": rows, "tokens": tokens, "context": context, "ragged": ragged, "norm": norm, "cap": cap,
            "window": window, "slopes": slopes, "prefix": prefix, **heads, **more}


def listed():
    return [
        # One conversation decoding: the smallest call, where the launch is what counts.
        _case("append-decode-b1", "append", M27, 1, 1, 1000, norm=True),
        # The headline verify step's batch (64 rows x 4 tokens, contexts up to 512).
        _case("append-verify-b64-k4", "append", M27, 64, 4, 512, norm=True),
        # A long prompt's chunk, begun inside a page.
        _case("append-prefill-2048", "append", M27, 1, 2048, 14341, norm=True),
        # A ragged batch of prompts in small pages, whole heads rotated, no norms.
        _case("append-ragged-b37", "append", G128, 37, 900, 700, ragged="all", page=16),
        # One conversation decoding over a short context: latency.
        _case("attend-decode-b1-1k", "attend", M27, 1, 1, 1000),
        # A serving batch decoding at medium context.
        _case("attend-decode-b64-8k", "attend", M27, 64, 1, 8192),
        # Speculative verify over long contexts.
        _case("attend-verify-b16-k4-32k", "attend", M27, 16, 4, 32768),
        # One token over a very long context, small pages.
        _case("attend-decode-b1-256k", "attend", G128, 1, 1, 262144, page=16),
        # The eighth chunk of a 16K prompt: the longest call.
        _case("attend-prefill-2048-16k", "attend", M27, 1, 2048, 14336),
        # One prompt's chunk beside 23 rows that decode, in one call.
        _case("attend-mixed-b24", "attend", G128, 24, 777, 4000, ragged="mixed", page=32),
        # A decoding batch of a model that caps its scores and looks back over a window.
        _case("attend-window-cap-b32", "attend", G128, 32, 1, 12000, cap=50.0, window=4096, page=128),
        # Prompts of a model that prefers near positions, heads of its own for every query, each prompt's prefix seen by all of it.
        _case("attend-slopes-prefix-b4", "attend", M64, 4, 1000, 500, ragged="all", slopes=True, prefix=700, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    heads = dict(rng.choice((M27, M27, G128, M64)), page=rng.choice((16, 32, 64, 128)))
    if rng.random() < 0.35:
        rows = _log(rng, 1, 64)
        tokens = rng.choice((1, rng.randint(2, 8), _log(rng, 9, 2048 // rows + 9)))
        ragged = rng.choice(("", "all")) if tokens > 1 else ""
        case = _case("", "append", heads, rows, tokens, _log(rng, 1, 8192 // rows + 100), ragged, rng.random() < 0.5)
    else:
        kind = rng.choice(("decode", "decode", "verify", "prefill", "mixed"))
        options = rng.choice(({}, {}, {}, {"cap": 30.0}, {"window": _log(rng, 16, 4096)}, {"slopes": True}, {"cap": 50.0, "slopes": True}))
        if kind == "prefill":
            rows, tokens = _log(rng, 1, 8), _log(rng, 20, 1024)
            context = rng.choice((0, _log(rng, 1, 8192 // rows)))
            if rng.random() < 0.25:
                options = {"prefix": context + rng.randint(1, tokens)}
            case = _case("", "attend", heads, rows, tokens // rows + 9, context, rng.choice(("", "all")), **options)
        elif kind == "mixed":
            rows = _log(rng, 2, 32)
            case = _case("", "attend", heads, rows, _log(rng, 20, 600), _log(rng, 10, 60000 // rows), "mixed", **options)
        else:
            rows = _log(rng, 1, 64)
            tokens = 1 if kind == "decode" else rng.randint(2, 8)
            case = _case("", "attend", heads, rows, tokens, _log(rng, 1, min(65536, 300000 // rows)), "", **options)
    del case["name"]
    return case


def _lengths(case):
    """(new tokens, first position) of each row: from the case alone."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    n, t, c = case["rows"], case["tokens"], case["context"]
    tokens = [t] + [t if not case["ragged"] else 1 if case["ragged"] == "mixed" else rng.randint(max(1, t // 8), t) for _ in range(n - 1)]
    return tokens, [c] + [rng.randint(c * 3 // 4, c) for _ in range(n - 1)]


def _sees(case, i, n):
    """How many positions the token at position i of a row of n positions sees."""
    return min(n, max(i + 1, case["prefix"])) - (max(0, i + 1 - case["window"]) if case["window"] else 0)


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    tokens, first = _lengths(case)
    total = sum(tokens)
    if case["op"] == "append":  # queries, keys, values and angles in; queries (16 bits), keys and values (8 bits), scales out
        touched = sum((p + t - 1) // case["page"] - p // case["page"] + 1 for t, p in zip(tokens, first))
        elements = total * (hq + 2 * hkv) * hd
        return {"bytes": elements * 2 + total * case["rot"] * 4 + total * (hq + hkv) * hd * 2 + touched * hkv * 2, "flops": 10 * elements}
    pairs = positions = 0
    for t, p in zip(tokens, first):
        n = p + t
        lo = max(0, p + 1 - case["window"]) if case["window"] else 0
        positions += n - lo
        pairs += sum(_sees(case, p + i, n) for i in range(t))
    return {"bytes": positions * hkv * (2 * hd + 2 / case["page"]) + total * hq * hd * 4, "flops": 4 * hd * hq * pairs}


def _gen(seed, name):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(name.encode())) & 0x7FFFFFFFFFFF)
    return g


def prepare(case, seed):
    rows, hq, hkv, hd, page = case["rows"], case["hq"], case["hkv"], case["hd"], case["page"]
    tokens, first = _lengths(case)
    ends = [(p + t + page - 1) // page for t, p in zip(tokens, first)]
    width, used = max(ends), sum(ends)
    count = used + 3  # some that no row holds
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    randn = lambda name, *shape: torch.randn(*shape, generator=_gen(seed, name), device="cuda", dtype=F32)  # noqa: E731
    ids = torch.randperm(count, generator=_gen(seed, "pages"), device="cuda").to(torch.int32)
    table = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
    at = 0
    for r, e in enumerate(ends):
        table[r, :e] = ids[at : at + e]
        at += e
    s = {"case": case, "position": ints(first), "table": table, "longest": max(tokens)}
    ragged = bool(case["ragged"])
    start = [0]
    for t in tokens:
        start.append(start[-1] + t)
    total = start[-1]
    s["start"] = ints(start) if ragged else None
    # Pages as a filled cache has them: normal values, the pages' magnitudes spread over powers of two.
    for name, shape in (("k", (count, hkv, page, hd)), ("v", (count, hkv, page // 16, hd, 16))):
        power = torch.randint(-2, 3, (count, hkv), generator=_gen(seed, name + "_scale"), device="cuda")
        x = randn(name, *shape).mul_(64.0).clamp_(-448.0, 448.0)
        s[name + "_pages"] = x.to(E4M3).view(torch.uint8)
        s[name + "_scale"] = (power + 121 if name == "v" else power.clamp(-1, 0) + 121).to(torch.uint8)
        del x
    if case["op"] == "attend":
        s["q"] = randn("q", total, hq, hd).mul_(2.0).to(BF16)
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=F32) / hq) if case["slopes"] else None
        s["prefix"] = ints([min(case["prefix"], p + t) for t, p in zip(tokens, first)]) if case["prefix"] else None
    else:
        # The projection's output: queries, keys and values of a token side by side, as a step's product leaves them.
        qkv = randn("qkv", total, hq + 2 * hkv, hd).mul_(1.5).to(BF16)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
        where = torch.tensor([p + i for t, p in zip(tokens, first) for i in range(t)], dtype=F64, device="cuda")
        angle = where[:, None] / THETA ** (torch.arange(0, case["rot"], 2, dtype=F64, device="cuda") / case["rot"])
        s["cos"], s["sin"] = (f(torch.cat((angle, angle), 1)).to(BF16) for f in (torch.cos, torch.sin))
        s["q_norm"], s["k_norm"] = ((randn(n, hd) * 0.1).to(BF16) for n in ("q_norm", "k_norm")) if case["norm"] else (None, None)
        # The pages that the call writes, and where in each its first new token comes.
        pages = [(r, j, max(0, p - j * page)) for r, (t, p) in enumerate(zip(tokens, first)) for j in range(p // page, (p + t - 1) // page + 1)]
        s["touched"] = table[[r for r, _, _ in pages], [j for _, j, _ in pages]].long()
        s["offset"] = torch.tensor([o for _, _, o in pages], device="cuda")
    # Each token's row and its number in it.
    s["row"] = torch.tensor([r for r, t in enumerate(tokens) for _ in range(t)], device="cuda")
    s["nth"] = torch.tensor([i for t in tokens for i in range(t)], device="cuda")
    return s


def run(s):
    append = s["case"]["op"] == "append"
    if not own:
        return _plain_append(s) if append else _plain_attend(s)
    sys.path.insert(0, os.path.join(os.getcwd(), "qwen38-27b-aws_amd")) if "qwen38_amd" not in sys.modules else None
    from qwen38_amd import ext

    c = s["case"]
    cache = ext.PagedCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if append:
        q = ext.paged_append(cache, s["new_k"], s["new_v"], s["position"], s["table"], cos=s["cos"], sin=s["sin"], q=s["q"],
                             q_start=s["start"], max_tokens=s["longest"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return _cache_values(s, q)
    return ext.paged_attention(cache, s["q"], s["position"], s["table"], q_start=s["start"], max_tokens=s["longest"], cap=c["cap"],
                               slopes=s["slopes"], window=c["window"], prefix=s["prefix"])


def _cache_values(s, q):
    """What an append leaves: the rotated queries, and the cache's bytes as the types that they are."""
    e8 = torch.float8_e8m0fnu
    return {"q": q, "k": s["k_pages"].view(E4M3), "v": s["v_pages"].view(E4M3), "k_scale": s["k_scale"].view(e8), "v_scale": s["v_scale"].view(e8)}


# --------------------------------------------------------------------------------------------------- the plain forms


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w.float())


def _rotated(x, cos, sin):
    rot = cos.shape[-1]
    a, rest = x[..., :rot], x[..., rot:]
    half = torch.cat((-a[..., rot // 2 :], a[..., : rot // 2]), -1)
    return torch.cat((a * cos.float()[:, None] + half * sin.float()[:, None], rest), -1)


def _plain_append(s):
    page = s["case"]["page"]
    q = _rotated(_normed(s["q"].float(), s["q_norm"]), s["cos"], s["sin"]).to(BF16)
    k = _rotated(_normed(s["new_k"].float(), s["k_norm"]), s["cos"], s["sin"])
    v = s["new_v"].float()
    # A token that is not finite: a key of NaN, a value of zero.
    fine = (torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))[..., None]
    position = s["position"].long()[s["row"]] + s["nth"]
    into, slot = s["table"][s["row"], position // page].long(), position % page
    _plain_code(s["k_pages"], s["k_scale"], torch.where(fine, k, 0.0), fine, s, (into, slice(None), slot))
    _plain_code(s["v_pages"], s["v_scale"], torch.where(fine, v, 0.0), fine | True, s, (into, slice(None), slot // 16, slice(None), slot % 16))
    return _cache_values(s, q)


def _plain_code(pages, scale, x, fine, s, where):
    """The new tokens x [tokens, hkv, hd] into the pages: the pages' new scales, what they held before coded again, the tokens."""
    page, touched, offset, into = s["case"]["page"], s["touched"], s["offset"], where[0]
    most = torch.zeros(scale.shape, dtype=F32, device=scale.device)
    most.scatter_reduce_(0, into[:, None].expand(-1, scale.shape[1]), x.abs().amax(-1), "amax")
    fraction, power = torch.frexp(most[touched])  # 448 is 0.875 x 2^9
    need = (power - 9 + (fraction > 0.875) + 127).clamp(1, 254)
    old = scale[touched].int()
    new = torch.where(offset[:, None] > 0, torch.maximum(old, need), need)
    scale[touched] = new.to(torch.uint8)
    held = pages[touched]
    before = torch.arange(page, device=held.device) < offset[:, None]  # [touched, page]
    before = before[:, None, :, None] if held.dim() == 4 else before.view(-1, 1, page // 16, 1, 16)
    factor = torch.exp2((old - new).float()).view(*new.shape, *[1] * (held.dim() - 2))
    pages[touched] = torch.where(before, (held.view(E4M3).float() * factor).to(E4M3).view(torch.uint8), held)
    inverse = torch.exp2(127.0 - scale[into].float())[..., None]
    pages[where] = torch.where(fine, x * inverse, float("nan")).to(E4M3).view(torch.uint8)


def _plain_attend(s):
    c = s["case"]
    rows, hq, hkv, hd, n = c["rows"], c["hq"], c["hkv"], c["hd"], s["longest"]
    ids = s["table"].long()
    times = lambda b: torch.exp2(b[ids].float() - 127.0)  # noqa: E731
    k = (s["k_pages"][ids].view(E4M3).float() * times(s["k_scale"])[..., None, None]).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [rows, hkv, S, hd]
    v = (s["v_pages"][ids].view(E4M3).float() * times(s["v_scale"])[..., None, None, None]).permute(0, 2, 1, 3, 5, 4).flatten(2, 4)
    size = k.shape[2]
    position = s["position"].long()
    total = position + torch.zeros_like(position).index_add_(0, s["row"], torch.ones_like(s["row"]))
    q = torch.zeros(rows, n, hq, hd, dtype=F32, device=k.device).index_put_((s["row"], s["nth"]), s["q"].float())
    q = q.view(rows, n, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(rows, hkv, -1, hd)
    x = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * hd**-0.5).view(rows, hkv, hq // hkv, n, size)
    del k
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    at = (position[:, None] + torch.arange(n, device=q.device))[:, :, None]  # [rows, n, 1]
    j = torch.arange(size, device=q.device)
    seen = (j <= at) if not c["prefix"] else (j <= at) | (j < s["prefix"][:, None, None])
    seen = seen & (j < total[:, None, None])
    if c["window"]:
        seen = seen & (j > at - c["window"])
    if c["slopes"]:
        x = x + s["slopes"].view(hkv, -1, 1, 1) * (j - at).float()[:, None, None]
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
    o = torch.matmul((w / w.sum(-1, keepdim=True)).view(rows, hkv, -1, size), v).view(rows, hkv, hq // hkv, n, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(rows, n, hq, hd)[s["row"], s["nth"]].to(BF16)


# --------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    tokens, first = _lengths(case)
    hq, hkv, hd, page = case["hq"], case["hkv"], case["hd"], case["page"]
    table = s["table"].tolist()
    worth = {n: s[n + "_pages"].view(E4M3).double() for n in ("k", "v")} if case["op"] == "append" else None
    at = 0
    if case["op"] == "append":
        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * (1.0 + w.double())
            half = case["rot"] // 2
            c, n = s["cos"].double()[:, None, :half], s["sin"].double()[:, None, :half]
            a, b = x[..., :half], x[..., half : 2 * half]
            return torch.cat((a * c - b * n, b * c + a * n, x[..., 2 * half :]), -1)

        q, k, v = turned(s["q"], s["q_norm"]), turned(s["new_k"], s["k_norm"]), s["new_v"].double()
        scales = {n: torch.exp2(s[n + "_scale"].double() - 127.0) for n in ("k", "v")}
        for r, (t, p) in enumerate(zip(tokens, first)):
            for j in range(p // page, (p + t - 1) // page + 1):
                lo, hi, e = max(p, j * page), min(p + t, (j + 1) * page), table[r][j]
                for n, x in (("k", k), ("v", v)):
                    x = x[at + lo - p : at + hi - p]
                    need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((0, 2)) / 448.0)))
                    old = scales[n][e].clone()
                    new = torch.maximum(old, need) if lo > j * page else need
                    scales[n][e] = new
                    body = worth[n][e]
                    by = body if n == "k" else body.transpose(-1, -2).reshape(hkv, page, hd)  # [hkv, page, hd]
                    by = by.clone()
                    by[:, : lo - j * page] *= (old / new)[:, None, None]
                    by[:, lo - j * page : hi - j * page] = x.transpose(0, 1) / new[:, None, None]
                    worth[n][e] = by if n == "k" else by.view(hkv, page // 16, 16, hd).transpose(-1, -2)
            at += t
        return {"q": q, "k": worth["k"], "v": worth["v"], "k_scale": scales["k"], "v_scale": scales["v"]}
    out = torch.empty(sum(tokens), hq, hd, dtype=F64, device="cuda")
    for r, (t, p) in enumerate(zip(tokens, first)):
        n, ids = p + t, s["table"][r, : (p + t + page - 1) // page].long()
        i = torch.arange(p, p + t, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= i) | (j < min(case["prefix"], n))
        if case["window"]:
            seen = seen & (i - j < case["window"])
        for h in range(hkv):
            k = (s["k_pages"][ids, h].view(E4M3).double() * torch.exp2(s["k_scale"][ids, h].double() - 127)[:, None, None]).reshape(-1, hd)[:n]
            v = s["v_pages"][ids, h].view(E4M3).double() * torch.exp2(s["v_scale"][ids, h].double() - 127)[:, None, None, None]
            v = v.transpose(-1, -2).reshape(-1, hd)[:n]
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = s["q"][at : at + t, g].double() @ k.t().contiguous() / math.sqrt(hd)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - float(s["slopes"][g]) * (i - j)
                out[at : at + t, g] = torch.softmax(x.masked_fill(~seen, float("-inf")), -1) @ v
        at += t
    return out
