"""``DecodeModel.run`` over the 8-bit paged cache: prompts and decode steps through whole layers (GPU).

Against transformers' own attention the cache's rounding shows: a code is off by 2^-4 of its value at most, 2^-4 /
sqrt(3) = 3.6% in the root mean square if errors are even over the step and less on average (a step spans values
of twice the size: 2.6%).  V's errors reach the output no larger than that, averaged over the keys; K's move the
scores by as much again.  The mean bar is therefore the bf16 cache's 1e-2 and 2.6% for each of K and V."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.helpers import errors, np_f32

pytestmark = pytest.mark.gpu

PAGE = 16


def i32(a, dev):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def build(pkg, dev, n_layers=2, n_pages=64, seed=3):
    from inference_server_amd import decode as dec

    cfg = dec.DecoderConfig(hidden=256, heads=8, kv_heads=2, experts=16, top_k=4, moe_intermediate=128)
    gen = torch.Generator(device=dev).manual_seed(seed)
    layers = [dec.DecoderLayerWeights.random(cfg, dev, gen) for _ in range(n_layers)]
    caches = [dec.PagedKVCacheFp8(n_layers, n_pages, cfg.kv_heads, dev) for _ in range(2)]
    return dec, cfg, gen, [dec.DecodeModel(cfg, layers, c) for c in caches]


STEPS = [[30, 0, 40], [1, 33, 1], [1, 1, 1], [0, 1, 20], [1, 1, 1]]


def test_graph_replays_match_eager_over_changing_lengths(pkg, dev):
    """Plan and layers of a step in one graph: prompts, a mixed step and decode steps, against the eager model on a
    cache of its own, to the bit, with eager work between the replays."""
    dec, cfg, gen, (eager, graphed) = build(pkg, dev)
    T, B, width = 72, 3, 12
    tables = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(5)).to(torch.int32).to(dev)
    graph, (g_h, g_cached, g_new, g_tables, g_free), g_out, g_plan = graphed.capture_run(
        torch.zeros((T, cfg.hidden), dtype=torch.bfloat16, device=dev), i32([0] * B, dev), i32([1] * B, dev), tables,
        free, 40)
    assert all((c.view(torch.uint8) == 0).all() for c in graphed.cache.k)  # capturing stored nothing
    cached, used = [0] * B, 0
    for new in STEPS:
        h = torch.randn((T, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
        rest = torch.cat([free[used:], free.new_full((used,), -1)])
        plan = eager.plan(i32(cached, dev), i32(new, dev), tables, rest, T, 40)
        out = eager.run(h, plan)
        for dst, src in ((g_h, h), (g_cached, i32(cached, dev)), (g_new, i32(new, dev)), (g_free, rest)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        assert torch.equal(out[:n], g_out[:n]) and torch.isfinite(out.float()).all()
        assert torch.equal(g_tables, tables) and torch.equal(g_plan.slots, plan.slots)
        for a, b in zip(eager.cache.k + eager.cache.v, graphed.cache.k + graphed.cache.v):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        used += plan.pages_used.item()
        cached = plan.context_lens.tolist()
    assert cached == [33, 36, 63]


def test_run_is_its_operators(pkg, dev):
    """One layer's ``run`` against the public operators called one by one, to the bit."""
    dec, cfg, gen, (model, other) = build(pkg, dev, n_layers=1)
    w, cache = model.layers[0], other.cache.layer(0)
    args = (i32([0, 0], dev), i32([21, 40], dev), torch.full((2, 4), -1, dtype=torch.int32, device=dev),
            torch.arange(64, dtype=torch.int32, device=dev))
    h = torch.randn((61, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
    plan = model.plan(*args, 61, 40)
    got = model.run(h, plan)
    qkv = torch.nn.functional.linear(pkg.rms_norm(h, w.ln1, cfg.rms_eps), w.wqkv)
    q = pkg.qk_norm_rope_append_fp8(qkv, w.q_norm, w.k_norm, model.inv_freq, cfg.heads, cfg.kv_heads, cfg.rms_eps, *cache,
                                    plan)
    a = pkg.paged_attention_fp8(q, *cache, plan, 128 ** -0.5)
    o = torch.nn.functional.linear(a.view(61, -1), w.wo)
    want = pkg.moe_sublayer_fp8(h, w.ln2, cfg.rms_eps, w.router, cfg.top_k, w.q13, w.s13, w.q2, w.s2, add=o)
    assert torch.equal(got, want)


def test_wrong_cache_is_refused(pkg, dev):
    dec, cfg, gen, (model, _) = build(pkg, dev, n_layers=1)
    h = torch.zeros((1, cfg.hidden), dtype=torch.bfloat16, device=dev)
    one = i32([1], dev)
    tables = torch.zeros((1, 2), dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        model.step(h, one, one, tables)
    bf16 = dec.DecodeModel(cfg, model.layers, dec.PagedKVCache(1, 4, cfg.kv_heads, dev))
    with pytest.raises(TypeError):
        bf16.run(h, model.plan(one, one, tables, one, 1, 1))


def test_attention_sublayer_matches_transformers(pkg, dev):
    """Prompts, then decode steps, through one layer's attention sublayer, fed transformers' own layer inputs."""
    transformers = pytest.importorskip("transformers")
    from tests.test_gpu_decode import _model
    from inference_server_amd import decode as dec

    cfg, hf = _model(dev, n_layers=1, heads=8, kv_heads=2, hidden=256)
    pkg.swap_moe_blocks(hf, quantize_fp8=True)
    H, lens, steps = cfg.hidden_size, [70, 33, 5], 3
    dcfg = dec.DecoderConfig(hidden=H, heads=8, kv_heads=2, experts=cfg.num_experts, top_k=cfg.num_experts_per_tok,
                             moe_intermediate=cfg.moe_intermediate_size, rms_eps=cfg.rms_norm_eps, rope_theta=1e6)
    w = dec.DecoderLayerWeights.from_hf_layer(hf.model.layers[0], dcfg)
    inv_freq = dec.default_inv_freq(dcfg, dev)
    cap = {}
    layer = hf.model.layers[0]
    layer.register_forward_pre_hook(
        lambda m, args, kw: cap.__setitem__("in", kw.get("hidden_states", args[0] if args else None)), with_kwargs=True)
    layer.self_attn.register_forward_hook(lambda m, args, out: cap.__setitem__("attn", out[0]))
    kv = dec.PagedKVCacheFp8(1, 40, 2, dev)
    tables = torch.full((len(lens), 8), -1, dtype=torch.int32, device=dev)
    free, used = torch.arange(39, -1, -1, dtype=torch.int32, device=dev), 0
    past = [transformers.DynamicCache() for _ in lens]
    cached = [0] * len(lens)
    for step in range(steps + 1):
        new = lens if step == 0 else [1] * len(lens)
        inputs, refs = [], []
        with torch.no_grad():
            for b, n in enumerate(new):
                ids = torch.randint(0, cfg.vocab_size, (1, n), device=dev)
                pos = torch.arange(cached[b], cached[b] + n, device=dev)[None]
                hf(input_ids=ids, position_ids=pos, past_key_values=past[b], use_cache=True)
                inputs.append(cap["in"].reshape(n, H))
                refs.append(cap["attn"].reshape(n, H))
            h = torch.cat(inputs).contiguous()
            plan = pkg.paged_plan(i32(cached, dev), i32(new, dev), tables, free[used:], sum(new), max(new), 8, 2)
            got = dec.attention_sublayer_fp8(w, h, plan, inv_freq, *kv.layer(0))
        used += plan.pages_used.item()
        cached = plan.context_lens.tolist()
        _, mean_rel = errors(np_f32(got), np_f32(torch.cat(refs)))
        assert mean_rel <= 1e-2 + 2 * 2.6e-2, (step, mean_rel)
        assert np.isfinite(np_f32(got)).all()
