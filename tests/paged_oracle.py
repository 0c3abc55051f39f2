"""The paged 8-bit cache and attention over it in 64 bits, position by position on the CPU: what include/q38.h says of
q38_paged_append and q38_paged_attention, for the tests."""

from __future__ import annotations

import math

import torch

F64, E4M3 = torch.float64, torch.float8_e4m3fn


def values(cache):
    """Keys and values [pages, kv_heads, page, hd] and their scales [pages, kv_heads] as float64 on the CPU."""
    k, v, ks, vs = (t.cpu() for t in cache)
    ks, vs = torch.exp2(ks.double() - 127), torch.exp2(vs.double() - 127)
    k = k.view(E4M3).double() * ks[..., None, None]
    v = v.view(E4M3).double().transpose(-1, -2).flatten(2, 3) * vs[..., None, None]
    return k, v, ks, vs


def norm_rotate(x, w, cos, sin, eps):
    x = x.cpu().double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1 + w.cpu().double())
    if cos is not None:
        half = cos.shape[1] // 2
        c, s = cos.cpu().double()[:, None], sin.cpu().double()[:, None]
        a, b = x[..., :half], x[..., half : 2 * half]
        x = torch.cat((a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:], x[..., 2 * half :]), -1)
    return x


def need(most):
    """The smallest power of two with values up to `most` (per head) within +-448 of it, at least 2^-126."""
    return torch.exp2(torch.ceil(torch.log2(most / 448)).clamp_min(-126))


def appended(cache, k, v, position, pages, starts, page):
    """(keys, values, key scales, value scales, written) after appending k, v [tokens, kv_heads, hd] (float64, normed and rotated):
    values as `values` gives them, the new ones not rounded; what the page held already as it is; written [pages, page]."""
    ks, vs, ksc, vsc = values(cache)
    written = torch.zeros(ks.shape[0], page, dtype=torch.bool)
    for r, p in enumerate(position):
        n = starts[r + 1] - starts[r]
        if p < 0 or not n:
            continue
        for j in range(p // page, (p + n - 1) // page + 1):
            if j >= pages.shape[1] or not 0 <= int(pages[r, j]) < ks.shape[0]:
                continue
            e, lo, hi = int(pages[r, j]), max(p, j * page), min(p + n, (j + 1) * page)
            new = slice(starts[r] + lo - p, starts[r] + hi - p)
            fine = (k[new].isfinite().all(-1) & v[new].isfinite().all(-1)).unsqueeze(-1)  # [tokens, kv_heads, 1]
            for held, scale, x, bad in ((ks, ksc, k[new], math.nan), (vs, vsc, v[new], 0.0)):
                s = need(torch.where(fine, x, 0.0).abs().amax((0, 2)))
                scale[e] = torch.maximum(scale[e], s) if lo > j * page else s
                held[e, :, lo - j * page : hi - j * page] = torch.where(fine, x, bad).transpose(0, 1)
            written[e, lo - j * page : hi - j * page] = True
    return ks, vs, ksc, vsc, written


def attention(cache, q, position, pages, starts, page, scale, cap=0.0, slopes=None, window=0, prefix=None):
    """(outputs, sums of weights x |values|) [tokens, q_heads, hd] in float64; tokens of no row are NaN."""
    k, v, _, _ = values(cache)
    count, hkv, _, hd = k.shape
    hq = q.shape[1]
    q = q.cpu().double()
    out, size = torch.full(q.shape, math.nan, dtype=F64), torch.full(q.shape, math.nan, dtype=F64)
    for r, p in enumerate(position):
        t0, n = starts[r], starts[r + 1] - starts[r]
        if p < 0:
            out[t0 : t0 + n], size[t0 : t0 + n] = 0, 0
            continue
        if not n:
            continue
        total = p + n
        ids = [int(pages[r, j]) if j < pages.shape[1] else -1 for j in range((total + page - 1) // page)]
        at = torch.tensor([e if 0 <= e < count else count for e in ids])
        keys = torch.cat((k, torch.full((1, *k.shape[1:]), math.nan, dtype=F64)))[at].transpose(1, 2).reshape(-1, hkv, hd)[:total]
        vals = torch.cat((v, torch.full((1, *v.shape[1:]), math.nan, dtype=F64)))[at].transpose(1, 2).reshape(-1, hkv, hd)[:total]
        i, j = torch.arange(p, total)[:, None], torch.arange(total)[None]
        seen = j <= i
        if prefix is not None:
            seen = seen | (j < prefix[r])
        if window:
            seen = seen & (j > i - window)
        for h in range(hq):
            g = h // (hq // hkv)
            s = q[t0 : t0 + n, h] @ keys[:, g].T * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s + float(slopes[h]) * (j - i)
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            val = vals[:, g]
            # A weight that is not there takes nothing from a value, NaN or not.
            clean = torch.where(val.isnan(), 0.0, val)
            lost = (seen.double() @ val.isnan().double()) > 0
            out[t0 : t0 + n, h] = torch.where(lost, math.nan, w @ clean)
            size[t0 : t0 + n, h] = w @ clean.abs()
    return out, size
