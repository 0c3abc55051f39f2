"""The paged 8-bit cache on the GPU: appending (norm, rotation, powers of two per page and head, e4m3) and attention over the
pages, against tests/paged_oracle.py in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as po
from qwen38_amd import ext

BF16, E4M3, EPS = torch.bfloat16, torch.float8_e4m3fn, 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen(seed)) * scale


def filled_cache(pages, hkv, hd, page, seed):
    """A cache of normal values, the pages' magnitudes over powers of two."""
    c = ext.paged_cache(pages, hkv, hd, page)
    for n, (t, s) in enumerate(((c.k, c.k_scale), (c.v, c.v_scale))):
        t.copy_((randn(seed + n, *t.shape) * 64).clamp(-448, 448).to(E4M3).view(torch.uint8))
        s.copy_(torch.randint(119, 124, s.shape, generator=gen(seed + 5 + n)).to(torch.uint8))
    return c


def table(pages, rows, width, seed):
    """Distinct pages for every row and place."""
    assert rows * width <= pages
    return torch.randperm(pages, generator=gen(seed))[: rows * width].reshape(rows, width).to(torch.int32)


def starts_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def angles(where, rot):
    a = torch.tensor(where, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.cat((a, a), 1)
    return a.cos().to(BF16), a.sin().to(BF16)


def dev(*ts):
    return tuple(None if t is None else t.cuda() for t in ts)


def clone(cache):
    return ext.PagedCache(*(t.clone() for t in cache))


def check_appended(cache, before, k, v, position, pages, starts, page):
    """The cache after an append against the oracle's from `before`: scales equal; new keys and values within half an e4m3 step (2^-4
    of the value, 2^-10 of the scale below e4m3's normal range) plus what float32 arithmetic adds (2^-20 of the page's largest);
    what the pages held as it was, within half a step of the new scale where that grew; all else byte for byte."""
    want = po.appended(before, k, v, position, pages, starts, page)
    got = po.values(cache)
    old = po.values(before)
    written = want[4]
    touched = written.any(1)
    for n, name in enumerate(("keys", "values")):
        x, y, scale, was = got[n], want[n], want[2 + n], old[2 + n]
        assert torch.equal(got[2 + n], scale), f"{name}: scales"
        s = scale[..., None, None]
        at = written[:, None, :, None].expand_as(x)
        bound = torch.maximum(y.abs() * 2**-4, s * 2**-10) + 448 * s * 2**-20
        assert torch.equal(x.isnan() & at, y.isnan() & at), f"{name}: NaN"
        off = ((x - y).abs() / bound)[at & ~y.isnan()]
        assert off.numel() == 0 or float(off.max()) <= 1, f"{name}: new ones off by {float(off.max())} of the bound"
        # The slots before a page's first new token (none if that is its first slot).
        before_new = (torch.arange(page)[None] < torch.where(touched, written.int().argmax(1), 0)[:, None])[:, None, :, None]
        grown = (scale > was)[..., None, None] & before_new
        held = grown.expand_as(x) & ~y.isnan()
        assert bool(((x - y).abs() <= torch.maximum(y.abs() * 2**-4, s * 2**-10))[held].all()), f"{name}: coded again"
        raw, raw_was = ((c.k if n == 0 else c.v.transpose(-1, -2).flatten(2, 3)).cpu() for c in (cache, before))
        same = ~at & ~grown
        assert torch.equal(raw[same], raw_was[same]), f"{name}: bytes that no token wrote"



APPENDS = [
    # heads q/kv, hd, rot, page, lengths, positions, norm
    (6, 2, 256, 64, 64, [1], [0], True),
    (24, 4, 256, 64, 64, [1, 1, 1], [63, 64, 200], True),
    (6, 1, 256, 64, 16, [4, 4], [14, 31], False),  # four tokens over the end of a page
    (8, 8, 64, 64, 32, [33, 1, 7, 0, 70], [0, 31, 95, 3, 17], False),
    (8, 2, 128, 128, 16, [257, 3], [5, 640], True),
    (4, 4, 64, 0, 128, [300, 129], [100, 127], False),  # no rotation
    (5, 5, 128, 40, 128, [128, 1], [128, 255], True),  # a page filled whole, an odd rotation
    (10, 2, 256, 256, 128, [200], [60], True),
    (3, 3, 64, 8, 64, [2, 2], [-1, 62], False),  # a row that is skipped
]


@pytest.mark.gpu
@pytest.mark.parametrize("hq, hkv, hd, rot, page, lengths, position, norm", APPENDS)
@pytest.mark.parametrize("grow", [1.0, 40.0])
def test_append(gpu, hq, hkv, hd, rot, page, lengths, position, norm, grow):
    rows, starts = len(lengths), starts_of(lengths)
    tokens = starts[-1] + 2  # two behind the last row
    width = max((max(p, 0) + n + page - 1) // page for p, n in zip(position, lengths)) + 1
    cache = filled_cache(rows * width + 3, hkv, hd, page, 1)
    pages = table(rows * width + 3, rows, width, 2)
    qkv = (randn(3, tokens, hq + 2 * hkv, hd) * 1.5).to(BF16)  # side by side, as a projection leaves them
    qkv[:, hq:] *= grow if not norm else 1.0
    qkv[:, hq + hkv :] *= grow if norm else 1.0
    q_norm, k_norm = ((randn(s, hd) * 0.2).to(BF16) for s in (4, 5)) if norm else (None, None)
    where = [max(p, 0) + i for p, n in zip(position, lengths) for i in range(n)] + [0, 0]
    cos, sin = angles(where, rot) if rot else (None, None)
    k = po.norm_rotate(qkv[:, hq : hq + hkv], k_norm, cos, sin, EPS)
    before = clone(cache)
    d = qkv.cuda()
    q_out = torch.full((tokens, hq, hd), 7.0, dtype=BF16, device="cuda")
    dc, ds, dq, dk, dp = dev(cos, sin, q_norm, k_norm, pages)
    ext.paged_append(cache, d[:, hq : hq + hkv], d[:, hq + hkv :], torch.tensor(position, dtype=torch.int32).cuda(), dp, cos=dc, sin=ds, q=d[:, :hq],
                     q_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_tokens=max(lengths), q_norm=dq, k_norm=dk, eps=EPS, q_out=q_out)
    check_appended(cache, before, k, qkv[:, hq + hkv :].double(), position, pages, starts, page)
    want = po.norm_rotate(qkv[:, :hq], q_norm, cos, sin, EPS)[: starts[-1]]
    got = q_out.double().cpu()
    # bf16's half step, and float32's over the norm and the rotation (their terms up to the head's largest).
    bound = want.abs() * 2**-8 + want.abs().amax(-1, keepdim=True) * 2**-19
    assert bool(((got[: starts[-1]] - want).abs() <= bound).all())
    assert bool((got[starts[-1] :] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd, page", [(64, 16), (256, 64), (128, 128)])
def test_appending_token_by_token_fills_the_page_as_one_call_does(gpu, hd, page):
    """With magnitudes that never grow past the first token's, the page's scale is the first token's all along."""
    n, hkv = page + 5, 2
    k, v = ((randn(s, n, hkv, hd).clamp(-2, 2)).to(BF16).cuda() for s in (1, 2))
    k[0, :, 0], v[0, :, 0] = 3.0, 3.0
    k[page, :, 0], v[page, :, 0] = 3.0, 3.0
    one, many = ext.paged_cache(3, hkv, hd, page), ext.paged_cache(3, hkv, hd, page)
    pages = torch.tensor([[2, 0]], dtype=torch.int32).cuda()
    at = lambda p: torch.tensor([p], dtype=torch.int32).cuda()  # noqa: E731
    ext.paged_append(one, k, v, at(0), pages)
    for i in range(n):
        ext.paged_append(many, k[i : i + 1], v[i : i + 1], at(i), pages)
    for a, b in zip(one, many):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_scale_that_grows_step_by_step_and_a_row_taken_back(gpu):
    """Each token 1.9 times the last: the scale grows with most of them, and what was held is coded again each time, each time
    exactly but for e4m3's subnormals. Then the row is taken back into the page: its scale stays."""
    hkv, hd, page = 1, 64, 32
    cache = ext.paged_cache(2, hkv, hd, page)
    pages = torch.tensor([[1]], dtype=torch.int32).cuda()
    x = torch.stack([torch.full((1, hd), 1.9**i) for i in range(20)]).to(BF16).cuda()
    for i in range(20):
        ext.paged_append(cache, x[i : i + 1], -x[i : i + 1], torch.tensor([i], dtype=torch.int32).cuda(), pages)
        k, v = ext.paged_values(cache)
        scale = 2.0 ** (int(cache.k_scale[1, 0]) - 127)
        assert scale == float(po.need(x[i].double().cpu().amax()))
        want = x[: i + 1, 0].float()
        bound = torch.maximum(want * 2**-4, torch.full_like(want, scale * 2**-9))  # subnormals: several roundings of half a step and halved
        assert bool(((k[1, 0, : i + 1] - want).abs() <= bound).all()) and bool(((v[1, 0, : i + 1] + want).abs() <= bound).all())
    grown = cache.k_scale.clone()
    ext.paged_append(cache, x[:1], x[:1], torch.tensor([7], dtype=torch.int32).cuda(), pages)
    assert torch.equal(cache.k_scale, grown)
    ext.paged_append(cache, x[:1], x[:1], torch.tensor([0], dtype=torch.int32).cuda(), pages)  # the page begun anew
    assert int(cache.k_scale[1, 0]) == int(math.log2(float(po.need(torch.ones(1).double())))) + 127


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["key", "value"])
def test_a_token_that_is_not_finite_is_seen_as_nan_and_harms_no_other(gpu, bad, where):
    hkv, hd, page, n = 2, 128, 32, 50
    k, v = ((randn(s, n, hkv, hd)).to(BF16).cuda() for s in (1, 2))
    q = randn(3, n, 4, hd).to(BF16).cuda()
    cache, clean = ext.paged_cache(4, hkv, hd, page), ext.paged_cache(4, hkv, hd, page)
    pages = torch.tensor([[3, 1]], dtype=torch.int32).cuda()
    zero = torch.zeros(1, dtype=torch.int32).cuda()
    ext.paged_append(clean, k, v, zero, pages)
    (k if where == "key" else v)[20, 1, 5] = bad
    ext.paged_append(cache, k, v, zero, pages)
    assert torch.equal(cache.k[:, 0], clean.k[:, 0]) and torch.equal(cache.v_scale[:, 0], clean.v_scale[:, 0])
    assert bool(ext.paged_values(cache)[0][3, 1, 20].isnan().all()) and bool((ext.paged_values(cache)[1][3, 1, 20] == 0).all())
    out = ext.paged_attention(cache, q, zero, pages)
    good = ext.paged_attention(clean, q, zero, pages)
    assert torch.equal(out[:, :2], good[:, :2])  # the other KV head
    assert bool(out[:20, 2:].isfinite().all()) and bool(out[20:, 2:].isnan().all())
    # A later row that has the token only behind its window sees nothing of it.
    late = ext.paged_attention(cache, q[:1], torch.tensor([40], dtype=torch.int32).cuda(), pages, window=20)
    assert bool(late.isfinite().all())


@pytest.mark.gpu
def test_zeros_and_tiny_and_huge_values(gpu):
    hkv, hd, page = 1, 64, 16
    cache = ext.paged_cache(3, hkv, hd, page)
    pages = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda()
    x = torch.zeros(3 * page, hkv, hd, dtype=BF16)
    x[page : 2 * page] = torch.finfo(BF16).tiny
    x[2 * page :] = 3e38
    ext.paged_append(cache, x.cuda(), x.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), pages)
    k, v = (t.cpu() for t in ext.paged_values(cache))
    assert bool((k[0] == 0).all()) and bool((v[0] == 0).all())
    for t in (k, v):
        assert bool(((t[2].double() / 3e38 - 1).abs() <= 2**-4 + 2**-8).all())  # 3e38 as a bf16, then e4m3
        assert bool(((t[1].double() / torch.finfo(BF16).tiny - 1).abs() <= 2**-4).all())


ATTENDS = [
    # heads q/kv, hd, page, lengths, positions, options
    (6, 1, 256, 64, [1], [0], {}),
    (24, 4, 256, 64, [1, 1, 1, 1], [0, 63, 64, 700], {}),
    (24, 4, 256, 64, [4, 4, 4], [0, 61, 333], {}),
    (12, 2, 256, 32, [8, 8], [120, 5], {}),
    (8, 8, 64, 16, [1, 1, 1], [15, 16, 1000], {}),
    (64, 1, 128, 16, [1, 1], [77, 400], {}),  # 64 query heads to one
    (7, 1, 64, 128, [3, 3], [126, 2000], {}),
    (10, 2, 128, 32, [1, 0, 33, 1], [400, 9, 0, 31], {}),  # an empty row among them
    (24, 4, 256, 64, [100], [0], {}),
    (12, 2, 256, 64, [130, 5], [77, 300], {}),
    (4, 4, 64, 32, [257], [3], {}),
    (16, 2, 128, 16, [90, 1, 1, 60], [10, 500, 0, 64], {}),
    (4, 2, 128, 64, [70, 1], [200, 300], {"cap": 20.0}),
    (8, 2, 64, 16, [1, 1, 1], [0, 40, 300], {"window": 17}),
    (8, 2, 256, 64, [90, 3], [200, 300], {"window": 1}),
    (8, 2, 128, 32, [150], [500], {"window": 64, "cap": 30.0}),
    (8, 8, 64, 64, [1, 70], [300, 100], {"slopes": True}),
    (6, 2, 128, 32, [40, 2], [30, 200], {"slopes": True, "cap": 10.0, "window": 50}),
    (8, 4, 64, 32, [100, 20, 1], [0, 50, 80], {"prefix": [60, 64, 0]}),
    (6, 1, 256, 64, [80], [20], {"prefix": [1000], "slopes": True}),  # past the row's end: all of it
    (6, 1, 256, 64, [2, 2], [-1, 20], {}),  # a row that is skipped
]


def attend_case(hq, hkv, hd, page, lengths, position, options, seed=1, q_scale=2.0):
    rows, starts = len(lengths), starts_of(lengths)
    width = max((max(p, 0) + n + page - 1) // page for p, n in zip(position, lengths)) + 1
    cache = filled_cache(rows * width + 3, hkv, hd, page, seed)
    pages = table(rows * width + 3, rows, width, seed + 20)
    q = (randn(seed + 30, starts[-1], hq, hd) * q_scale).to(BF16)
    slopes = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).float() if options.get("slopes") else None
    prefix = torch.tensor(options["prefix"], dtype=torch.int32) if "prefix" in options else None
    more = {"cap": options.get("cap", 0.0), "window": options.get("window", 0)}
    uniform = len(set(lengths)) == 1
    dq, dp, dsl, dpf = dev(q, pages, slopes, prefix)
    call = dict(q_start=None if uniform else torch.tensor(starts, dtype=torch.int32).cuda(), max_tokens=None if uniform else max(lengths),
                slopes=dsl, prefix=dpf, **more)
    args = (cache, dq, torch.tensor(position, dtype=torch.int32).cuda(), dp)
    want = po.attention(cache, q, position, pages, starts, page, hd**-0.5, slopes=slopes, prefix=None if prefix is None else prefix.tolist(), **more)
    return args, call, want


def check_attention(got, want):
    """bf16's half step of the output (2^-8); of every weight (2^-8 of its share in the sum of weights x |values|); and 2^-13 of that sum
    for float32 scores and exponentials."""
    out, size = want
    got = got.double().cpu()
    assert torch.equal(got.isnan(), out.isnan())
    bound = out.abs() * 2**-8 + size * (2**-8 + 2**-13) + 1e-30
    off = torch.where(out.isnan(), 0.0, (got - out).abs() / bound)
    print(f"largest {float(off.max()):.3f} of the bound", flush=True)
    assert float(off.max()) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("hq, hkv, hd, page, lengths, position, options", ATTENDS)
def test_attention(gpu, hq, hkv, hd, page, lengths, position, options):
    args, call, want = attend_case(hq, hkv, hd, page, lengths, position, options)
    check_attention(ext.paged_attention(*args, **call), want)
