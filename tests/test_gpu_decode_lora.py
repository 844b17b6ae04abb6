"""``DecodeModel`` with adapters and ``OutputHead``: prompts and single tokens of many adapters through whole layers, and
the log probabilities they end in (GPU)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

L, RANK = 5, 32


def i32(a, dev):
    return torch.tensor(a, dtype=torch.int32, device=dev)


def build(pkg, dev, n_layers=2, cache="fp8", seed=3, std=0.05):
    from inference_server_amd import decode as dec

    cfg = dec.DecoderConfig(hidden=256, heads=8, kv_heads=2, experts=16, top_k=4, moe_intermediate=128)
    gen = torch.Generator(device=dev).manual_seed(seed)
    layers = [dec.DecoderLayerWeights.random(cfg, dev, gen) for _ in range(n_layers)]
    adapters = [dec.LayerAdapters.empty(cfg, L, RANK, dev) for _ in range(n_layers)]
    randn = lambda *s: (torch.randn(s, generator=gen, device=dev) * std).to(torch.bfloat16)  # noqa: E731
    for a in adapters:
        for i, r in enumerate([8, 32, 16, 5]):  # the last one is not loaded
            a.qkv.load(i, [(randn(r, a.qkv.in_features), randn(n, r)) for n in a.qkv.columns], 2.0)
            a.o.load(i, [(randn(r, a.o.in_features), randn(cfg.hidden, r))], 1.0)
    make = (lambda: dec.PagedKVCacheFp8(n_layers, 64, cfg.kv_heads, dev)) if cache == "fp8" else \
        (lambda: dec.PagedKVCache(n_layers, 64, cfg.kv_heads, dev))
    return dec, cfg, gen, lambda: dec.DecodeModel(cfg, layers, make(), adapters)


def step_args(dev, new, T):
    return (i32([0] * len(new), dev), i32(new, dev), torch.full((len(new), 8), -1, dtype=torch.int32, device=dev),
            torch.arange(64, dtype=torch.int32, device=dev), T, max(new))


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1, 1], [40, 3, 1, 60, 17, 9], [100, 90, 80, 120, 70, 1]])
def test_rows_have_their_own_adapter_alone(pkg, dev, new):
    """A sequence's rows are, to the bit, what they are when every sequence has that adapter; without one, those of a model
    without adapters."""
    dec, cfg, gen, model = build(pkg, dev)
    T = sum(new) + 5  # some padding
    ids = [2, -1, 0, 3, 4, 1]
    h = torch.randn((T, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)

    def run(adapters):
        m = model()
        plan = m.plan(*step_args(dev, new, T))
        return m.run(h, plan, None if adapters is None else m.lora_plan(i32(adapters, dev), plan))

    mixed, plain, at = run(ids), run(None), 0
    for n, i in zip(new, ids):
        rows = slice(at, at + n)
        want = run([i] * len(ids)) if i >= 0 else plain
        assert torch.equal(mixed[rows], want[rows])
        assert torch.equal(mixed[rows], plain[rows]) == (i in (-1, 4))
        at += n


def test_an_adapter_is_what_it_merges_to(pkg, dev):
    """Against a model whose weights have the adapter added.  The two round at different places, so k and v are up to a
    bf16 step, 2^-8 of their value, apart, which moves a share of 2^-8 / 2^-3 of the cache's e4m3 codes by one of their
    steps, 2^-3 of the value at most: 2^-5.5 = 2.2% in the root mean square, for K and for V (whose share reaches the
    output no larger than that); 1e-2 for the rest."""
    dec, cfg, gen, model = build(pkg, dev, n_layers=1)
    new = [30, 1, 50]
    T = sum(new)
    h = torch.randn((T, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
    m = model()
    plan = m.plan(*step_args(dev, new, T))
    got = dec.attention_sublayer_fp8(m.layers[0], h, plan, m.inv_freq, *m.cache.layer(0), m.adapters[0],
                                     m.lora_plan(i32([1, 1, 1], dev), plan))
    other = model()
    w, pools = other.layers[0], other.adapters[0]

    def merged(weight, pool):
        out, at = weight.float().clone(), 0
        for p, n in enumerate(pool.columns):
            a, b = pool.a[1, p * RANK:(p + 1) * RANK].float(), pool.b[1, at:at + n].float()
            out[at:at + n] += pool.scales[1] * b @ a
            at += n
        return out.to(torch.bfloat16)

    w2 = dec.DecoderLayerWeights(cfg, w.ln1, merged(w.wqkv, pools.qkv), w.q_norm, w.k_norm, merged(w.wo, pools.o), w.ln2, w.router,
                                 w.q13, w.s13, w.q2, w.s2)
    plan2 = other.plan(*step_args(dev, new, T))
    want = dec.attention_sublayer_fp8(w2, h, plan2, other.inv_freq, *other.cache.layer(0)).float()
    base = dec.attention_sublayer_fp8(w, h, plan2, other.inv_freq, *other.cache.layer(0)).float()
    bar = (1e-2 + 2 * 2.0 ** -5.5) * want.abs().mean()
    assert (got.float() - want).abs().mean() <= bar < 0.5 * (base - want).abs().mean()


def test_replays_follow_lengths_and_adapters(pkg, dev):
    """Plans, layers and adapters of a step in one graph, prompts and decode steps, against the eager model to the bit."""
    dec, cfg, gen, model = build(pkg, dev)
    eager, graphed = model(), model()
    T, B = 72, 3
    tables = torch.full((B, 12), -1, dtype=torch.int32, device=dev)
    free = torch.arange(64, dtype=torch.int32, device=dev)
    graph, (g_h, g_cached, g_new, g_tables, g_free, g_ids), g_out, g_plan = graphed.capture_run(
        torch.zeros((T, cfg.hidden), dtype=torch.bfloat16, device=dev), i32([0] * B, dev), i32([1] * B, dev), tables, free, 40,
        adapter_ids=i32([-1] * B, dev))
    cached, used = [0] * B, 0
    for new, ids in (([30, 0, 40], [0, 1, 2]), ([1, 33, 1], [3, 1, -1]), ([1, 1, 1], [0, 0, 0]), ([1, 1, 1], [4, 3, 2])):
        h = torch.randn((T, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
        rest = torch.cat([free[used:], free.new_full((used,), -1)])
        plan = eager.plan(i32(cached, dev), i32(new, dev), tables, rest, T, 40)
        out = eager.run(h, plan, eager.lora_plan(i32(ids, dev), plan))
        for dst, src in ((g_h, h), (g_cached, i32(cached, dev)), (g_new, i32(new, dev)), (g_free, rest), (g_ids, i32(ids, dev))):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        assert torch.equal(out[:n], g_out[:n]) and torch.isfinite(out[:n].float()).all()
        used += plan.pages_used.item()
        cached = plan.context_lens.tolist()


def test_steps_over_the_bf16_cache(pkg, dev):
    """``step`` and its capture with adapters: rows as with that adapter alone, replays as the eager step."""
    dec, cfg, gen, model = build(pkg, dev, cache="bf16")
    B, ids = 6, [2, -1, 0, 3, 4, 1]
    h = torch.randn((B, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
    pos = torch.zeros(B, dtype=torch.int32, device=dev)
    tables = torch.arange(B, dtype=torch.int32, device=dev)[:, None].contiguous()
    run = lambda m, a: m.step(h, pos, pos + 1, tables, **({} if a is None else {"lora": m.lora_plan(i32(a, dev))}))  # noqa: E731
    mixed, plain = run(model(), ids), run(model(), None)
    for b, i in enumerate(ids):
        want = plain if i < 0 else run(model(), [i] * B)
        assert torch.equal(mixed[b], want[b])
    m = model()
    graph, statics, out = m.capture(h, pos, pos + 1, tables, adapter_ids=i32([0] * B, dev))
    for a in (ids, ids[::-1], [-1] * B):
        statics[4].copy_(i32(a, dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(model(), a))


@pytest.mark.parametrize("vocab", [512, 1000])
def test_from_hidden_states_to_log_probabilities(pkg, dev, vocab):
    """A step of several adapters, the head behind it, and the given tokens' log probabilities: those of the head's own
    logits in 64 bits."""
    dec, cfg, gen, model = build(pkg, dev)
    new, ids = [25, 1, 40], [1, 3, -1]
    T = sum(new)
    h = torch.randn((T, cfg.hidden), generator=gen, device=dev).to(torch.bfloat16)
    m = model()
    plan = m.plan(*step_args(dev, new, T))
    out = m.run(h, plan, m.lora_plan(i32(ids, dev), plan))
    head = dec.OutputHead(torch.ones(cfg.hidden, dtype=torch.bfloat16, device=dev),
                          (torch.randn((vocab, cfg.hidden), generator=gen, device=dev) * 0.1).to(torch.bfloat16))
    tokens = torch.randint(0, vocab, (T,), generator=gen, device=dev)
    for rows in (slice(0, T), slice(0, 3)):  # the library's linear kernel, and its own
        x = out[rows].contiguous()
        logits = head.logits(x)
        r = head.token_logprobs(x, tokens[rows], 4)
        y = pkg.rms_norm(x, head.norm, head.eps).double() @ head.weight.double().T
        assert (logits.double() - y).abs().max() <= 2.0 ** -8 * y.abs().max() + 1e-4
        want = torch.log_softmax(logits.double(), 1)
        assert (r.logprobs.double() - want.gather(1, tokens[rows, None])[:, 0]).abs().max() <= 1e-5
        assert torch.equal(r.top_ids, torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :4])
