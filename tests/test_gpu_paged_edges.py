"""The paged operators on the GPU where they can go wrong: scores that leap, pages that are not there, bytes that no token wrote, rows
skipped, empty and very many, work cut in parts, every number of query row tiles, other streams, captured graphs, pools past 4 GiB;
and appending and attending together. Against tests/paged_oracle.py in 64 bits, with test_gpu_paged's bounds."""

from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as po
from qwen38_amd import ext
from test_gpu_paged import BF16, E4M3, angles, attend_case, check_attention, clone, dev, filled_cache, gen, randn, starts_of, table


def attend(cache, q, position, pages, starts, *, uniform=False, want=None, slopes=None, prefix=None, **options):
    """The operator against the oracle; returns its outputs."""
    lengths = [b - a for a, b in zip(starts, starts[1:])]
    page, hd = cache.k.shape[2:]
    if want is None:
        want = po.attention(cache, q, position, pages, starts, page, hd**-0.5, slopes=slopes, prefix=prefix, **options)
    dq, dp, dsl, dpos = dev(q, pages, slopes, torch.tensor(position, dtype=torch.int32))
    got = ext.paged_attention(cache, dq, dpos, dp, q_start=None if uniform else torch.tensor(starts, dtype=torch.int32).cuda(),
                              max_tokens=None if uniform else max(lengths), slopes=dsl,
                              prefix=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda(), **options)
    check_attention(got, want)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("tokens, context", [(1, 900), (9, 500), (70, 900), (300, 3000)])
def test_scores_that_leap(gpu, hd, tokens, context):
    """One key in a row's first page, and one in its last, is far nearer to every query than all others: scores of some 46 (66 in
    powers of two), found after thousands of small ones, and before. Sums of |q k| stay below 100, where float32 scores are good to 100 x
    2^-22, a fifth of the bound's 2^-13."""
    page, hq, hkv = 32, 4, 2
    width = (context + tokens + page - 1) // page
    for place in (5, context - 1):
        cache = filled_cache(width, hkv, hd, page, 1)
        cache.k_scale.fill_(127 - 9)
        sign = torch.where(randn(2, hd) > 0, 1.0, -1.0)
        pages = table(width, 1, width, 3)
        far = int(pages[0, place // page])
        k = randn(7, hkv, page, hd, scale=8.0)
        k[:, place % page] = sign * 46 / math.sqrt(hd) * 2**5  # sign . key / sqrt(hd) = 46
        cache.k[far] = k.to(E4M3).view(torch.uint8).cuda()
        cache.k_scale[far] = 127 - 5
        q = (sign + 0.1 * randn(4, tokens, hq, hd)).to(BF16)
        attend(cache, q, [context], pages, [0, tokens], uniform=True)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("tokens", [2, 100])
@pytest.mark.parametrize("options", [{}, {"window": 40}])
def test_pages_that_are_not_there(gpu, hd, tokens, options):
    """Ids below zero and past the pool, and positions past the table: NaN for whoever sees them, and for nobody else."""
    page, rows = 32, 6
    cache = filled_cache(rows * 8, 2, hd, page, 1)
    position = [130, 130, 130, 8 * page - tokens // 2, 9 * page, 2**30]
    pages = table(rows * 8, rows, 8, 2)
    pages[0, 1], pages[1, 2], pages[2, (130 + tokens - 1) // page] = -1, rows * 8, -(2**31)
    q = randn(3, rows * tokens, 4, hd).to(BF16)
    starts = [tokens * r for r in range(rows + 1)]
    # The oracle's lists end with the row: a position far past the table is one just past it.
    want = po.attention(cache, q, [min(p, 9 * page) for p in position], pages, starts, page, hd**-0.5, **options)
    got = attend(cache, q, position, pages, starts, uniform=True, want=want, **options)
    assert bool(got[5 * tokens :].isnan().all())
    if options:
        assert bool(got[: 2 * tokens].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("hd, page", [(64, 128), (128, 16), (256, 64)])
@pytest.mark.parametrize("tokens", [1, 80])
def test_bytes_that_nobody_may_see_may_be_nan(gpu, hd, page, tokens):
    """NaN codes behind a row's last position, before its window, and in every page of nobody's."""
    position = [5, 200, 333]
    rows, width = len(position), (333 + tokens) // page + 2
    pages = table(rows * width, rows, width, 2)
    for window in (0, 50):
        cache = filled_cache(rows * width, 2, hd, page, 1)
        hide = torch.ones(rows * width, page, dtype=torch.bool)
        for r, p in enumerate(position):
            for j in range(max(0, p + 1 - window) if window else 0, p + tokens):
                hide[pages[r, j // page], j % page] = False
        cache.k.copy_(torch.where(hide[:, None, :, None].cuda(), 0x7F, cache.k))
        v = hide.view(rows * width, 1, page // 16, 1, 16).cuda()
        cache.v.copy_(torch.where(v, 0xFF, cache.v))
        for t in cache[2:]:
            t[hide.all(1).cuda()] = 255
        got = attend(cache, randn(3, rows * tokens, 4, hd).to(BF16), position, pages, [tokens * r for r in range(rows + 1)], uniform=True, window=window)
        assert bool(got.isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lengths, position", [
    ([0, 70, 0, 5, 0, 33], [3, 10, -1, 0, 0, -1]), ([0, 1, 0, 2], [9, 0, 0, -5]), ([40, 0, 1, 0, 300], [-1, 50, 600, 0, 200])])
def test_rows_skipped_and_empty_ones_and_the_tokens_behind(gpu, hd, lengths, position):
    starts, rows = starts_of(lengths), len(lengths)
    width = max(max(p, 0) + n for p, n in zip(position, lengths)) // 32 + 1
    cache, pages = filled_cache(rows * width, 2, hd, 32, 1), table(rows * width, rows, width, 2)
    behind = 7
    q = randn(3, starts[-1] + behind, 8, hd).to(BF16)
    out = torch.full_like(q, 5.0).cuda()
    dq, dp = dev(q, pages)
    ext.paged_attention(cache, dq, torch.tensor(position, dtype=torch.int32).cuda(), dp, q_start=torch.tensor(starts, dtype=torch.int32).cuda(),
                        max_tokens=max(lengths), out=out)
    want = po.attention(cache, q[: starts[-1]], position, pages, starts, 32, hd**-0.5)
    check_attention(out[: starts[-1]], want)
    assert bool((out[starts[-1] :] == 5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd, hq, hkv", [(64, 4, 1), (128, 2, 2), (256, 6, 1)])
@pytest.mark.parametrize("options", [{}, {"window": 700}, {"cap": 5.0, "slopes": True}, {"prefix": [100000]}])
def test_tiles_cut_in_parts(gpu, hd, hq, hkv, options):
    """Few query rows over many positions: workgroups share tiles, and join their parts."""
    for tokens, context in ((70 * 6 // (hq // hkv), 5000), (600, 2111)):
        args, call, want = attend_case(hq, hkv, hd, 64, [tokens], [context], options)
        got = ext.paged_attention(*args, **call)
        check_attention(got, want)
        assert torch.equal(got.view(torch.int16), ext.paged_attention(*args, **call).view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 3, 7, 10, 11])
@pytest.mark.parametrize("options", [{}, {"window": 100, "cap": 8.0}, {"slopes": True, "prefix": [0, 500, 90]}])
def test_every_number_of_query_row_tiles(gpu, hd, tokens, options):
    """6 query heads to a KV head: 6 to 66 query rows, one to four tiles of 16, and past them."""
    args, call, want = attend_case(12, 2, hd, 32, [tokens] * 3, [0, 480, 1500], options)
    check_attention(ext.paged_attention(*args, **call), want)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hq, hkv", [(64, 1), (98, 2), (33, 1)])
def test_many_query_heads_to_a_key_head(gpu, hd, hq, hkv):
    """33, 49 and 64 of them, with one and two tokens a row, alike and not."""
    for lengths, position in (([1, 1], [700, 3]), ([2, 2], [0, 90]), ([1, 2, 0, 1], [5, 300, 9, 44])):
        args, call, want = attend_case(hq, hkv, hd, 32, lengths, position, {})
        check_attention(ext.paged_attention(*args, **call), want)


@pytest.mark.gpu
@pytest.mark.parametrize("hd, hq, hkv", [(64, 2, 1), (256, 64, 1), (128, 5, 5)])
def test_many_rows(gpu, hd, hq, hkv):
    """More rows than a wave has lanes, short and long ones and none among them."""
    g = gen(1)
    lengths = torch.randint(0, 4, (150,), generator=g).tolist()
    for r in (0, 63, 64, 100, 149):
        lengths[r] = 40
    position = torch.randint(-3, 90, (150,), generator=g).tolist()
    args, call, want = attend_case(hq, hkv, hd, 16, lengths, position, {})
    check_attention(ext.paged_attention(*args, **call), want)


@pytest.mark.gpu
@pytest.mark.parametrize("hd, hq, hkv", [(64, 6, 1), (128, 8, 2), (256, 12, 2)])
@pytest.mark.parametrize("lengths", [[4, 4, 200, 4, 4], [4, 90, 7, 1, 0, 8], [1, 1, 1, 100], [10, 11, 12, 100], [100, 4, 30, 30]])
def test_rows_of_a_few_tokens_beside_a_long_one(gpu, hd, hq, hkv, lengths):
    """The rows that stream are chosen by the others' usual number of tokens: some fit, some do not."""
    args, call, want = attend_case(hq, hkv, hd, 32, lengths, [(97 * r) % 700 for r in range(len(lengths))], {})
    check_attention(ext.paged_attention(*args, **call), want)
    more = {**call, "max_tokens": sum(lengths)}  # a bound that no row comes near
    check_attention(ext.paged_attention(*args, **more), want)


@pytest.mark.gpu
def test_many_rows_of_one_token_and_a_long_row(gpu):
    args, call, want = attend_case(2, 1, 64, 128, [1] * 200, [(37 * r) % 3000 for r in range(200)], {})
    check_attention(ext.paged_attention(*args, **call), want)
    args, call, want = attend_case(4, 1, 64, 128, [1], [70000], {})
    check_attention(ext.paged_attention(*args, **call), want)


@pytest.mark.gpu
def test_rows_that_share_a_prefix(gpu):
    cache, pages = filled_cache(40, 2, 128, 32, 1), table(40, 3, 12, 2)
    pages[1, :6], pages[2, :6] = pages[0, :6], pages[0, :6]
    q = randn(3, 3 * 50, 4, 128).to(BF16)
    attend(cache, q, [200, 230, 250], pages, [0, 50, 100, 150], uniform=True)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_a_pool_past_4_gib(gpu, hd):
    """Pages at the end of a pool whose keys alone take more than 2^32 bytes give what the same pages give in a small one, appended to
    and attended over."""
    page, hkv, rows, width, tokens = 128, 8, 2, 5, 60
    count = 2**32 // (page * hkv * hd) + 64
    ids = count - 1 - torch.arange(rows * width).reshape(rows, width).to(torch.int32) * 3
    small, big = filled_cache(rows * width, hkv, hd, page, 1), ext.paged_cache(count, hkv, hd, page)
    mine = torch.arange(rows * width).reshape(rows, width).to(torch.int32)
    for a, b in zip(big, small):
        a[ids.flatten().long().cuda()] = b
    k, v, q = dev(randn(2, rows * tokens, hkv, hd).to(BF16), randn(3, rows * tokens, hkv, hd).to(BF16), randn(4, rows * tokens, hkv * 2, hd).to(BF16))
    position = torch.tensor([400, 555], dtype=torch.int32).cuda()
    out = []
    for cache, pages in ((small, mine.cuda()), (big, ids.cuda())):
        ext.paged_append(cache, k, v, position, pages)
        out.append((ext.paged_attention(cache, q, position, pages), ext.paged_attention(cache, q[:rows], position, pages)))
    for a, b in zip(*out):
        assert torch.equal(a, b) and bool(a.isfinite().all())
    for a, b in zip(big, small):
        assert torch.equal(a[ids.flatten().long().cuda()], b)
    del big
    torch.cuda.empty_cache()


def step(cache, t, position, pages, **options):
    q = ext.paged_append(cache, t["k"], t["v"], position, pages, cos=t["cos"], sin=t["sin"], q=t["q"], k_norm=t["norm"])
    return q, ext.paged_attention(cache, q, position, pages, **options)


def step_tensors(rows, tokens, hq, hkv, hd, seed):
    cos, sin = angles(list(range(rows * tokens)), hd // 2)
    fused = randn(seed, rows * tokens, (hq + 2 * hkv) * hd).to(BF16).cuda()
    cut = lambda a, n: fused[:, a * hd : (a + n) * hd].unflatten(1, (n, hd))  # noqa: E731
    return {"q": cut(0, hq), "k": cut(hq, hkv), "v": cut(hq + hkv, hkv), "cos": cos.cuda(), "sin": sin.cuda(), "norm": randn(seed + 1, hd).to(BF16).cuda()}


@pytest.mark.gpu
@pytest.mark.parametrize("hd, page, hq, hkv", [(128, 16, 4, 2), (256, 64, 6, 1), (64, 128, 2, 2)])
def test_appending_and_attending_as_a_sequence_is_served(gpu, hd, page, hq, hkv):
    """A prompt in two chunks, then tokens in ones and fours, two rows at a time, from one fused projection: each call's outputs
    against the oracle's over the bytes that the appends left, and those against the unquantized keys and values."""
    rows, width = 2, 512 // page
    cache, pages = ext.paged_cache(rows * width, hkv, hd, page), table(rows * width, rows, width, 1)
    for t in cache[:2]:
        t.fill_(0x7F)  # no initial contents are needed
    at = [0, 7]
    for n, tokens in enumerate((7, 150, 33, 1, 1, 4, 1, 4)):
        t = step_tensors(rows, tokens, hq, hkv, hd, 10 * n)
        dpos, dp = torch.tensor(at, dtype=torch.int32).cuda(), pages.cuda()
        if n == 0:  # row 1's first tokens by themselves
            first = step_tensors(1, 7, hq, hkv, hd, 5)
            step(cache, first, dpos[:1] * 0, dp[1:])
        before = clone(cache)
        q, got = step(cache, t, dpos, dp)
        starts = [0, tokens, 2 * tokens]
        check_attention(got, po.attention(cache, q, at, pages, starts, page, hd**-0.5))
        k = po.norm_rotate(t["k"], t["norm"], t["cos"], t["sin"], 1e-6)
        want = po.appended(before, k, t["v"].cpu().double(), at, pages, starts, page)
        now = po.values(cache)
        for x, y, s in ((now[0], want[0], want[2]), (now[1], want[1], want[3])):
            new = want[4][:, None, :, None].expand_as(x)
            bound = torch.maximum(y.abs() * 2**-4, s[..., None, None] * 2**-10) + 448 * s[..., None, None] * 2**-20
            assert bool(((x - y).abs() <= bound)[new].all())
        at = [p + tokens for p in at]


@pytest.mark.gpu
def test_on_another_stream(gpu):
    t = step_tensors(3, 40, 4, 2, 128, 1)
    pages, position = table(30, 3, 10, 1).cuda(), torch.tensor([0, 200, 33], dtype=torch.int32).cuda()
    one, other = filled_cache(30, 2, 128, 32, 1), filled_cache(30, 2, 128, 32, 1)
    want = step(one, t, position, pages)[1]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(other, t, position, pages)[1]
    side.synchronize()
    assert torch.equal(got, want)
    for a, b in zip(one, other):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, context", [(1, 300), (4, 1000), (60, 100), (200, 1500)])
def test_captured_and_replayed(gpu, tokens, context):
    """Two graphs of append and attention, each with its own scratch, replayed in turn over positions that move on, with eager work
    between, against eager calls from the same bytes."""
    hq, hkv, hd, page, rows = 6, 2, 128, 32, 2
    width = (context + 6 * tokens) // page + 1
    pages = table(rows * width, rows, width, 1).cuda()
    cache = filled_cache(rows * width, hkv, hd, page, 1)
    t = step_tensors(rows, tokens, hq, hkv, hd, 2)
    position = torch.tensor([context, context // 2], dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        step(clone(cache), t, position, pages)  # loads the kernels
        side.synchronize()
    for options in ({}, {"window": 77}):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(cache, t, position, pages, **options)[1])
        graphs.append(graph)
    eager = clone(cache)
    for n in range(6):
        want = step(eager, t, position, pages, **({"window": 77} if n % 2 else {}))[1]
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[n % 2], want), n
        for a, b in zip(cache, eager):
            assert torch.equal(a, b), n
        _ = torch.ones(1 << 20, device="cuda").sum().item()
        position += tokens
        t["k"].copy_(randn(50 + n, *t["k"].shape).to(BF16))


@pytest.mark.gpu
def test_what_is_refused_on_a_device(gpu):
    cache, pages, position = ext.paged_cache(8, 2, 64, 16), table(8, 2, 4, 1).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    q = torch.zeros(4, 4, 64, dtype=BF16).cuda()
    kv = torch.zeros(4, 2, 64, dtype=BF16).cuda()
    for call in (
        lambda: ext.paged_attention(cache, q.transpose(0, 1), position, pages),
        lambda: ext.paged_attention(cache, q.float(), position, pages),
        lambda: ext.paged_attention(cache, q[:3], position, pages),  # three tokens of two rows
        lambda: ext.paged_attention(cache, q, position.long(), pages),
        lambda: ext.paged_attention(cache, q, position, pages.t()),
        lambda: ext.paged_attention(cache, q, position, pages, q_start=position),
        lambda: ext.paged_attention(cache, q, position, pages, q_start=torch.zeros(3, dtype=torch.int32).cuda()),
        lambda: ext.paged_attention(cache, q, position, pages, slopes=torch.ones(4)),
        lambda: ext.paged_attention(cache._replace(v=cache.k), q, position, pages),
        lambda: ext.paged_append(cache, kv[:, :1], kv, position, pages),
        lambda: ext.paged_append(cache, kv, kv, position, pages, cos=torch.zeros(4, 64, dtype=BF16).cuda()),
        lambda: ext.paged_append(cache, kv, kv, position, pages, q_norm=torch.zeros(64, dtype=BF16).cuda()),
        lambda: ext.paged_append(cache, kv.transpose(1, 2), kv, position, pages),
        lambda: ext.paged_attention(cache, q, position, pages, window=2**32 + 5),
        lambda: ext.paged_attention(cache, q, position, pages, window=-1),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ext.paged_attention(cache, q, position, pages, window=3, prefix=position),
                 lambda: ext.paged_attention(cache, q, position, pages, scale=-1.0),
                 lambda: ext.paged_attention(cache, q, position, pages, scratch=torch.empty(1, dtype=torch.uint8).cuda()),
                 lambda: ext.paged_append(cache, kv, kv, position, pages, cos=torch.zeros(4, 12, dtype=BF16).cuda(), sin=torch.zeros(4, 12, dtype=BF16).cuda())):
        with pytest.raises(RuntimeError):
            call()
