"""The paged cache's refusals, before any device work: the C entries with pointers that are never read, the Python ones with host
tensors; and the 64-bit oracle's softmax weights against differences of its outputs."""

from __future__ import annotations

import ctypes

import pytest
import torch

import paged_oracle as po
from qwen38_amd import ext

P = 4096  # a device pointer that nothing reads


def args(**changes):
    c = ext._CacheArgs(P, P, P, P, 8, 2, 128, 32)
    r = ext._RowArgs(P, P, P, 3, 4, 10, 5)
    t = ext._TokenArgs()
    t.k = t.v = t.q = t.q_out = t.cos = t.sin = P
    t.k_token, t.k_head, t.v_token, t.v_head, t.q_token, t.q_head = 256, 128, 256, 128, 512, 128
    t.q_heads, t.rotary_dim, t.eps = 4, 64, 1e-6
    q = ext._QueryArgs(P, P, 4, 0.1, 0.0, 0)
    for name, value in changes.items():
        of, field = name.split("__")
        setattr({"c": c, "r": r, "t": t, "q": q}[of], field, value)
    return c, r, t, q


def error(rc):
    assert rc != 0
    return ext.library().q38_last_error().decode()


BOTH = [
    ({"c__k": None}, "null"), ({"c__v_scale": None}, "null"), ({"r__position": None}, "null"), ({"r__pages": None}, "null"),
    ({"c__head_dim": 96}, "head_dim"), ({"c__page_size": 48}, "page_size"), ({"c__page_size": 256}, "page_size"), ({"c__pages": 0}, "positive"),
    ({"c__kv_heads": 0}, "positive"), ({"c__k": P + 8}, "aligned"), ({"c__v": P + 4}, "aligned"), ({"r__rows": 0}, "positive"),
    ({"r__max_tokens": 0}, "positive"), ({"r__tokens": -1}, "positive"), ({"r__max_tokens": 11}, "above tokens"),
    ({"r__q_start": None}, "without q_start"), ({"r__max_pages": 1 << 26}, "2.30 positions"),
    ({"r__rows": 1 << 22, "r__tokens": 1 << 20}, "too large"),
]


@pytest.mark.parametrize("changes, message", BOTH)
def test_both_refuse_a_cache_or_rows_they_do_not_take(changes, message):
    lib, ref = ext.library(), ctypes.byref
    c, r, t, q = args(**changes)
    import re

    assert re.search(message, error(lib.q38_paged_append(ref(c), ref(r), ref(t), None)))
    assert re.search(message, error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P, 1 << 60, None)))


@pytest.mark.parametrize("changes, message", [
    ({"t__k": None}, "null"), ({"t__v": None}, "null"), ({"t__cos": None}, "null"), ({"t__q_out": None}, "go together"), ({"t__q": None}, "go together"),
    ({"t__q_heads": 0}, "q_heads"), ({"t__rotary_dim": 12}, "rotary_dim"), ({"t__rotary_dim": 136}, "rotary_dim"), ({"t__rotary_dim": -8}, "rotary_dim"),
    ({"t__k_token": 258}, "strides"), ({"t__q_head": 129}, "strides"), ({"t__v": P + 2}, "aligned"), ({"t__eps": -1.0}, "eps"),
    ({"t__eps": float("nan")}, "eps"),
])
def test_append_refuses(changes, message):
    lib, ref = ext.library(), ctypes.byref
    c, r, t, _ = args(**changes)
    assert message in error(lib.q38_paged_append(ref(c), ref(r), ref(t), None))


@pytest.mark.parametrize("changes, message", [
    ({"q__q": None}, "null"), ({"q__out": None}, "null"), ({"q__q_heads": 5}, "q_heads"), ({"q__q_heads": 130}, "q_heads"), ({"q__q_heads": 0}, "q_heads"),
    ({"q__scale": float("nan")}, "scale"), ({"q__scale": float("inf")}, "scale"), ({"q__scale": 0.0}, "scale"), ({"q__scale": -1.0}, "scale"), ({"q__cap": -1.0}, "cap"), ({"q__cap": float("inf")}, "cap"),
    ({"q__window": -1}, "window"), ({"q__window": 4, "q__prefix": P}, "exclude"), ({"q__out": P + 8}, "aligned"),
])
def test_attention_refuses(changes, message):
    lib, ref = ext.library(), ctypes.byref
    c, r, _, q = args(**changes)
    assert message in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P, 1 << 60, None))


def test_host_tensors_and_wrong_shapes_are_refused():
    cache = ext.paged_cache(2, 1, 64, 16, device="cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ext.paged_append(cache, x, x, i, i[None]), lambda: ext.paged_attention(cache, x, i, i[None])):
        with pytest.raises(ValueError, match="on a device"):
            call()
    with pytest.raises(ValueError, match="q must be"):
        ext.paged_attention(cache, x[0], i, i[None])
    with pytest.raises(ValueError, match="must be contiguous torch.int32"):
        ext._want("position", i.long(), torch.int32, (1,), -1)
    with pytest.raises(ValueError, match="must be contiguous torch.int32"):
        ext._want("position", i, torch.int32, (2,), -1)
    with pytest.raises(ValueError, match="last dim"):
        ext._heads_of("k", torch.zeros(1, 64, 64, dtype=torch.bfloat16).transpose(1, 2), 1, 64, -1)
    with pytest.raises(ValueError, match="k must be"):
        ext._heads_of("k", x.float(), 1, 64, -1)


def test_paged_values_reads_what_the_oracle_reads():
    g = torch.Generator().manual_seed(1)
    cache = ext.paged_cache(3, 2, 64, 32, device="cpu")
    for t in cache[:2]:
        t.copy_(torch.randint(0, 256, t.shape, generator=g).to(torch.uint8))
    for t in cache[2:]:
        t.copy_(torch.randint(100, 140, t.shape, generator=g).to(torch.uint8))
    for a, b in zip(ext.paged_values(cache), po.values(cache)[:2]):
        assert torch.equal(a.double().isnan(), b.isnan()) and torch.equal(a.double().nan_to_num(), b.nan_to_num())


def test_an_engine_sizes_its_paged_caches_and_refuses_others():
    from qwen38_amd.config import tiny_config

    cfg = tiny_config(1)  # layers 0-2 gated delta, 3 attention; MTP layer 4
    hkv = cfg.num_key_value_heads
    h = ext.Handle(cfg, 4, 4, 128, True, prefill_chunk=64, kv_cache_format="fp8", kv_pages=40, kv_page_size=32)
    for layer in (3, 4):
        assert h.buffer_size("self_attn.k_cache", layer) == h.buffer_size("self_attn.v_cache", layer) == 40 * hkv * 32 * 256
        assert h.buffer_size("self_attn.k_scale", layer) == h.buffer_size("self_attn.v_scale", layer) == 40 * hkv
    assert h.buffer_size("page_table", -1) == 4 * 4 * 4
    with pytest.raises(RuntimeError, match="no buffer"):
        ext.Handle(cfg, 4, 4, 128, True).buffer_size("page_table", -1)
    for changes, message in (({"kv_pages": -1}, "negative"), ({"kv_page_size": 48}, "kv_page_size"), ({"kv_page_size": 256}, "kv_page_size"),
                             ({"max_seq_len": 160, "kv_page_size": 128}, "multiple of kv_page_size"), ({"kv_cache_format": "bf16"}, "FP8")):
        kw = {"max_seq_len": 128, "kv_cache_format": "fp8", "kv_pages": 8, "kv_page_size": 64, **changes}
        with pytest.raises(RuntimeError, match=message):
            ext.Handle(cfg, 4, 4, kw.pop("max_seq_len"), True, **kw)


def test_calls_too_large_for_a_grid_are_refused():
    lib, ref = ext.library(), ctypes.byref
    c, r, t, q = args(c__kv_heads=4, q__q_heads=4, r__rows=1 << 16, r__tokens=1 << 17, r__max_tokens=2)
    assert "rows * kv_heads too large" in error(lib.q38_paged_append(ref(c), ref(r), ref(t), None))
    assert "rows * kv_heads too large" in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P, 1 << 60, None))
    assert lib.q38_paged_attention_scratch(ref(c), ref(r), 4) == 0
    c, r, t, q = args(c__kv_heads=16, q__q_heads=1024, r__rows=1, r__tokens=1 << 22, r__max_tokens=1 << 22)
    assert "query rows too many" in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P, 1 << 60, None))
    assert lib.q38_paged_attention_scratch(ref(c), ref(r), 1024) == 0


@pytest.mark.parametrize("changes, message", [
    ({"t__cos": P + 4}, "aligned"), ({"t__sin": P + 2}, "aligned"), ({"t__q_norm": P + 4}, "aligned"), ({"t__k_norm": P + 2}, "aligned")])
def test_append_refuses_misaligned_vectors(changes, message):
    c, r, t, _ = args(**changes)
    assert message in error(ext.library().q38_paged_append(ctypes.byref(c), ctypes.byref(r), ctypes.byref(t), None))


def test_a_scratch_that_is_too_small_or_misaligned_is_refused():
    lib, ref = ext.library(), ctypes.byref
    for changes in ({}, {"r__max_tokens": 10}):
        c, r, _, q = args(**changes)
        need = lib.q38_paged_attention_scratch(ref(c), ref(r), 4)
        assert need > 0
        assert "scratch is smaller" in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P, need - 1, None))
        assert "scratch is smaller" in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), None, need, None))
        assert "256-byte" in error(lib.q38_paged_attention(ref(c), ref(r), ref(q), P + 128, need, None))
