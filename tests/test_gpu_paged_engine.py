"""An engine over paged 8-bit caches (`Engine(kv_pages=...)`) on the GPU: its steps against the operators by themselves, against an
engine of the same weights over bf16 slabs, and a captured speculative step against its launches."""

from __future__ import annotations

import pytest
import torch

import paged_oracle as po
from qwen38_amd import ext, synth
from qwen38_amd.config import tiny_config, with_layers
from qwen38_amd.generate import batch_step_inputs, mtp_prefill_inputs, mtp_step_inputs, prefill_inputs, verify_inputs
from qwen38_amd.steps import Engine, MTPStep, StepGraph
from scenario import SPEC, spec_start, spec_states, steer_head
from spec_check import DeviceStep

BF16 = torch.bfloat16
B, K, S, CHUNK, PAGE, EACH = 3, 4, 256, 64, 32, 8


@pytest.fixture(scope="module")
def weights():
    cfg = with_layers(tiny_config(1), ("full_attention",))
    return cfg, dict((sp.name, v) for sp, v in synth.make_all(synth.model_specs(cfg), 5))


def paged(cfg, values, pages=None, **changes):
    e = Engine(cfg, B, K, S, prefill_chunk=CHUNK, kv_cache_format="fp8", kv_pages=B * EACH + 2, kv_page_size=PAGE, **changes)
    e.load(values.items())
    order = torch.randperm(B * EACH + 2, generator=torch.Generator().manual_seed(3)).tolist() if pages is None else pages
    for b in range(B):
        e.set_pages(b, order[b * EACH : (b + 1) * EACH])
    return e


def embeds(seed, *shape):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 0.02).to(BF16)


def steps(cfg, engine, probe=None):
    """Two prefill chunks of row 1 and one of row 2, two verify steps (row 0 idle in the first, and not all tokens kept), a decode
    step, the drafter's prefill and step; the outputs of rows that are active and tokens that are there."""
    step, mtp = StepGraph(engine), MTPStep(engine)
    h, out = cfg.hidden_size, []
    for n, (slot, start, valid) in enumerate(((1, 0, CHUNK), (1, CHUNK, 37), (2, 0, 5))):
        x = embeds(10 + n, 1, CHUNK, h)
        out.append(step(inputs_embeds=x, **prefill_inputs(cfg, slot, start, valid, CHUNK, BF16))[0, :valid])
        mtp(embeds(20 + n, 1, CHUNK, h), x, **mtp_prefill_inputs(cfg, slot, start, valid, CHUNK, BF16))
    for n, (pos, active, accepted) in enumerate((([0, 101, 5], [0, 1, 1], [0, 0, 0]), ([0, 103, 9], [1, 1, 1], [0, 2, 4]))):
        if probe:
            probe("before")
        v = verify_inputs(cfg, pos, K, S, BF16, active, accepted)
        got = step(inputs_embeds=embeds(30 + n, B, K, h), **v)
        if probe:
            probe("verify", v)
        on = [b for b in range(B) if active[b]]
        out.append(got[on].flatten(0, 1))
    d = batch_step_inputs(cfg, [4, 107, 13], S, BF16, [1, 0, 1])
    out.append(step(inputs_embeds=embeds(40, B, 1, h), **d)[[0, 2]].flatten(0, 1))
    m = mtp_step_inputs(cfg, [0, 90, 4], K, S, BF16, [0, 1, 1])
    out.append(mtp(embeds(50, B, K, h), embeds(51, B, K, h), **m)[1:].flatten(0, 1))
    torch.cuda.synchronize()
    return out


@pytest.mark.gpu
def test_verify_calls_are_the_operators(gpu, weights):
    """From each verify call's own projection: the layer's cache bytes are the standalone append's, and the o projection's input the
    standalone attention's output times bf16(sigmoid(gate)) in e5m2; the hardware sigmoid may round a gate to the next bf16 value
    (its error is some 2^-22, a bf16 step 2^-8: one in thousands), which an e5m2 code may pass on as one step."""
    cfg, values = weights
    engine = paged(cfg, values)
    engine.enable_probe(0)
    hq, hkv, hd = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    held = {}

    def probe(what, v=None):
        torch.cuda.synchronize()
        cache = engine.paged_cache(0)
        if what == "before":
            held["cache"] = ext.PagedCache(*(t.clone() for t in cache))
            return
        p = engine.probe(0)
        x = p["projection"]
        qg = x[:, : hq * hd * 2].view(-1, hq, 2, hd)
        k, val = (t.reshape(-1, hkv, hd) for t in x[:, hq * hd * 2 :].chunk(2, 1))
        position = torch.where(v["active"] > 0.5, v["position"], -1).to(torch.int32).cuda()
        q = ext.paged_append(held["cache"], k, val, position, engine.page_table, cos=v["cos"].reshape(B * K, -1).cuda(),
                             sin=v["sin"].reshape(B * K, -1).cuda(), q=qg[:, :, 0], q_norm=engine.buffer("self_attn.q_norm", 0).view(BF16),
                             k_norm=engine.buffer("self_attn.k_norm", 0).view(BF16), eps=cfg.rms_norm_eps)
        for name, a, b in zip(cache._fields, cache, held["cache"]):
            assert torch.equal(a, b), name
        o = ext.paged_attention(cache, q, position, engine.page_table)
        want = (o * torch.sigmoid(qg[:, :, 1].float()).to(BF16)).flatten(1).to(torch.float8_e5m2)
        on = (v["active"] > 0.5).repeat_interleave(K)
        got, want = p["mid"].to(torch.float8_e5m2).view(torch.uint8).cpu()[on].int(), want.view(torch.uint8).cpu()[on].int()
        off = got != want
        print(f"{int(off.sum())} of {off.numel()} gated codes differ", flush=True)
        assert float(off.float().mean()) <= 1e-3 and bool(((got - want).abs()[off] == 1).all())

    steps(cfg, engine, probe)


@pytest.mark.gpu
def test_the_steps_follow_an_engine_over_bf16_slabs(gpu, weights):
    """The caches: the slab engine's bf16 keys and values (of the same projections, where the calls see the same inputs: the one
    decoder layer's, and the drafter's) in e4m3, half a step of it (2^-4) and the slab's own roundings (2^-8 each) and, at the
    bottom of the range, 2^-10 of the page's scale apart. The hidden states: embeddings of 0.02 leave the layer's own output almost all of
    them; 8-bit keys and values move the attention by a few hundredths, and the next inputs' e5m2 rounding (2^-3) passes part of
    that on; 2^-2 by token in the norm is far below what a wrong page, row or position does (order one)."""
    cfg, values = weights
    engine = paged(cfg, values)
    slab = Engine(cfg, B, K, S, prefill_chunk=CHUNK)
    slab.load(values.items())
    for n, (a, b) in enumerate(zip(steps(cfg, engine), steps(cfg, slab))):
        off = (a.float() - b.float()).norm(dim=-1) / b.float().norm(dim=-1)
        print(f"call {n}: largest {float(off.max()):.4f}", flush=True)
        assert float(off.max()) <= 0.25
    table = engine.page_table.cpu()
    # The positions that calls wrote and no padding of a chunk did (the slab engine keeps that).
    written = {0: [(0, 0, 5), (1, 0, 101), (1, 103, 107), (2, 0, 5), (2, 9, 14)], engine.mtp_layer: [(1, 0, 94), (2, 0, 4)]}
    for layer, runs in written.items():
        k, v, ks, vs = po.values(engine.paged_cache(layer))
        for n, (x, s, y) in enumerate(((k, ks, slab.get_kv(layer)[0]), (v, vs, slab.get_kv(layer)[1]))):
            for row, lo, hi in runs:
                at = torch.arange(lo, hi)
                page = table[row, at // PAGE].long()
                got, want, scale = x[page, :, at % PAGE], y[row, :, lo:hi].double().cpu().transpose(0, 1), s[page]
                bound = want.abs() * (2**-4 + 2**-7) + scale[..., None] * 2**-10
                if n == 0:
                    # The slab's rotation a cos - b sin rounds a, b and both products to bf16: 2 x 2^-8 (|a| + |b|), which stays where
                    # the products cancel; a^2 + b^2 = x^2 + y^2 of the rotated pair, so |a| + |b| <= 2 max(|x|, |y|).
                    pair = want[..., : cfg.rotary_dim].abs().unflatten(-1, (2, -1)).amax(-2).repeat(1, 1, 2)
                    bound[..., : cfg.rotary_dim] += pair * 2**-6
                # A page whose scale grew later has been rounded twice: half a step of the last scale more.
                bound = bound + torch.maximum(want.abs() * 2**-4, scale[..., None] * 2**-10)
                off = float(((got - want).abs() / bound).max())
                print(f"layer {layer} {'kv'[n]} row {row} {lo}:{hi}: {off:.3f} of the bound", flush=True)
                assert off <= 1


@pytest.mark.gpu
def test_which_pages_a_row_has_does_not_matter(gpu, weights):
    cfg, values = weights
    one, other = steps(cfg, paged(cfg, values)), steps(cfg, paged(cfg, values, list(range(B * EACH))))
    for a, b in zip(one, other):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_decode_step_is_a_verify_of_one_token(gpu, weights):
    cfg, values = weights
    a, b = (Engine(cfg, B, 1, S, kv_cache_format="fp8", kv_pages=B * EACH, kv_page_size=PAGE) for _ in range(2))
    for e in (a, b):
        e.load(values.items())
    for n in range(PAGE + 3):
        d = batch_step_inputs(cfg, [n, 2 * n, 0], S, BF16, [1, 1, 0])
        x = embeds(60 + n, B, 1, cfg.hidden_size)
        one = StepGraph(a)(inputs_embeds=x, **d)
        two = StepGraph(b)(inputs_embeds=x, accepted=torch.ones(B, dtype=torch.int32), **d)
        assert torch.equal(one[:2], two[:2]), n
    for x, y in zip(a.paged_cache(0), b.paged_cache(0)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_rows_share_the_pages_of_a_prefix(gpu, weights):
    """A chunk prefilled into row 1 is row 2's too once row 2's table names its pages: both rows' next tokens give the same."""
    cfg, values = weights
    e = paged(cfg, values)
    step = StepGraph(e)
    step(inputs_embeds=embeds(70, 1, CHUNK, cfg.hidden_size), **prefill_inputs(cfg, 1, 0, CHUNK, CHUNK, BF16))
    mine, theirs = e.page_table[1].tolist(), e.page_table[2].tolist()
    e.set_pages(2, mine[: CHUNK // PAGE] + theirs[CHUNK // PAGE :])
    x = embeds(71, 1, K, cfg.hidden_size).expand(B, K, -1).contiguous()
    got = step(inputs_embeds=x, **verify_inputs(cfg, [0, CHUNK, CHUNK], K, S, BF16, [0, 1, 1], [0, 0, 0]))
    assert torch.equal(got[1], got[2]) and bool(got[1].isfinite().all())


@pytest.mark.gpu
def test_a_row_without_a_page_is_not_a_number_and_harms_no_other(gpu, weights):
    cfg, values = weights
    e, whole = paged(cfg, values), paged(cfg, values)
    e.set_pages(1, e.page_table[1].tolist()[:1])
    x = embeds(80, B, K, cfg.hidden_size)
    v = verify_inputs(cfg, [0, PAGE - 2, 3], K, S, BF16, [1, 1, 1], [0, 0, 0])
    got, want = StepGraph(e)(inputs_embeds=x, **v), StepGraph(whole)(inputs_embeds=x, **v)
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[1, :2], want[1, :2])
    assert bool(got[1, 2:].isnan().all())


@pytest.mark.gpu
def test_graph_replays_of_the_speculative_step_equal_its_launches(gpu):
    cfg = tiny_config(1)
    values = steer_head(dict((sp.name, v) for sp, v in synth.make_all(synth.model_specs(cfg), SPEC["seed"])), cfg, SPEC["seed"])
    b, s = SPEC["batch"], SPEC["max_seq_len"]
    states, _ = spec_states(cfg)
    engines = []
    for _ in range(2):
        e = Engine(cfg, b, SPEC["tokens"], s, mtp=True, kv_cache_format="fp8", kv_pages=b * s // 16, kv_page_size=16)
        e.load(values.items())
        for i, kind in enumerate(cfg.layer_types):
            if kind == "linear_attention":
                e.set_gdn(i, states[i])
        for layer in [*(i for i, kind in enumerate(cfg.layer_types) if kind != "linear_attention"), e.mtp_layer]:
            g = torch.Generator().manual_seed(layer)
            c = e.paged_cache(layer)
            for t, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
                t.copy_((torch.randn(t.shape, generator=g) * 32).to(torch.float8_e4m3fn).view(torch.uint8))
                scale.fill_(122)
        engines.append(e)
    start = spec_start(cfg)
    eager, graph = DeviceStep(engines[0], start), DeviceStep(engines[1], start)
    for n in range(SPEC["steps"]):
        print(f"step {n}", flush=True)
        eager()
        graph(graph=True)
        _ = torch.ones(1024, device="cuda").sum().item()  # eager work between replays
        for name in ("drafts", "picks", "match", "accepted", "position", "index", "hidden"):
            assert torch.equal(getattr(eager, name), getattr(graph, name)), (n, name)
    for layer in [*(i for i, kind in enumerate(cfg.layer_types) if kind != "linear_attention"), engines[0].mtp_layer]:
        for x, y in zip(engines[0].paged_cache(layer), engines[1].paged_cache(layer)):
            assert torch.equal(x, y), layer


@pytest.mark.gpu
def test_what_an_engine_refuses(gpu, weights):
    cfg, values = weights
    e = paged(cfg, values)
    for call in (lambda: e.get_kv(0), lambda: e.set_kv_scales(0, torch.ones(1), torch.ones(1)), lambda: e.set_pages(B, [0]),
                 lambda: e.set_pages(0, [B * EACH + 2]), lambda: e.set_pages(0, [-1]), lambda: e.set_pages(0, list(range(EACH + 1))),
                 lambda: e.set_pages(0, [5, 5])):
        with pytest.raises(ValueError):
            call()
    slab = Engine(cfg, B, K, S, kv_cache_format="fp8")
    with pytest.raises(ValueError):
        slab.paged_cache(0)
    with pytest.raises(ValueError):
        slab.set_pages(0, [0])


@pytest.mark.gpu
def test_a_loaded_model_decodes_over_pages(gpu, weights):
    """`runner.load` with kv_pages: a prompt prefilled in chunks and decoded greedily, its rows' pages given as they are needed, is the
    engine's whose rows had all theirs from the start."""
    from qwen38_amd import runner

    cfg, values = weights
    kw = dict(cfg=cfg, batch_size=B, max_seq_len=S, verify_tokens=1, chunk=CHUNK, weight_format="e4m3", kv_cache_format="fp8", kv_page_size=PAGE,
              log=lambda m: None)
    one, other = (runner.load(weights=((n, v) for n, v in values.items() if not n.startswith("mtp.")), kv_pages=B * EACH, **kw) for _ in range(2))
    free = list(range(B * EACH))[::-1]
    held = [[] for _ in range(B)]
    for r in range(B):
        other.engine.set_pages(r, [])

    def grow(row, tokens):
        while len(held[row]) * PAGE < tokens:
            held[row].append(free.pop())
        other.engine.set_pages(row, held[row])

    prompt = torch.randint(0, cfg.vocab_size, (CHUNK + 9,), generator=torch.Generator().manual_seed(9)).tolist()
    ids = []
    for model in (one, other):
        out = []
        for start in (0, CHUNK):
            part = prompt[start : start + CHUNK]
            if model is other:
                grow(1, start + len(part))
            x = torch.zeros(1, CHUNK, cfg.hidden_size, dtype=BF16, device="cuda")
            x[0, : len(part)] = values["embed_tokens"][part].cuda()
            h = model.prefill(inputs_embeds=x, **prefill_inputs(cfg, 1, start, len(part), CHUNK, BF16))[:, len(part) - 1 : len(part)]
        at = len(prompt)
        for _ in range(PAGE + 2):
            token = model.head.next_tokens(h.expand(B, -1, -1).contiguous())[1]
            out.append(token)
            if model is other:
                grow(1, at + 1)
            x = values["embed_tokens"][[token]].cuda().expand(B, -1).unsqueeze(1).contiguous()
            h = model.step(inputs_embeds=x, **batch_step_inputs(cfg, [0, at, 0], S, BF16, [0, 1, 0]))[1:2]
            at += 1
        ids.append(out)
        assert bool(h.isfinite().all())
    assert ids[0] == ids[1]


@pytest.mark.gpu
def test_pages_need_the_8_bit_format(gpu, weights):
    with pytest.raises(RuntimeError, match="FP8"):
        Engine(weights[0], B, K, S, kv_pages=8)
