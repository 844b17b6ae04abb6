"""``DecodeModel`` on the CPU: which caches its calls take (the layers' kernels are stand-ins)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


@pytest.fixture
def dec(pkg):
    from inference_server_amd import decode

    return decode


def model(dec, cache):
    layers = [SimpleNamespace(wqkv=torch.zeros(1)) for _ in range(2)]
    return dec.DecodeModel(dec.DecoderConfig(), layers, cache)


def test_step_takes_any_cache_with_k_and_v(dec, monkeypatch):
    seen = []
    monkeypatch.setattr(dec, "attention_sublayer", lambda w, h, pos, ctx, tables, inv_freq, k, v: seen.append((k, v)) or h)
    m = model(dec, SimpleNamespace(k=["k0", "k1"], v=["v0", "v1"]))
    assert m.step(torch.ones(1), None, None, None, moe=False).item() == 4.0
    assert seen == [("k0", "v0"), ("k1", "v1")]


def test_step_without_attention_needs_no_cache(dec, monkeypatch):
    monkeypatch.setattr(dec, "moe_sublayer", lambda w, h, o=None: h + 1)
    for cache in (None, dec.PagedKVCacheFp8(2, 1, 1, "cpu")):
        assert model(dec, cache).step(torch.ones(1), None, None, None, attention=False).item() == 3.0


def test_each_cache_has_its_calls(dec):
    fp8 = model(dec, dec.PagedKVCacheFp8(2, 1, 1, "cpu"))
    with pytest.raises(TypeError, match="PagedKVCacheFp8"):
        fp8.step(torch.ones(1), None, None, None)
    for cache in (dec.PagedKVCache(2, 1, 1, "cpu"), None):
        with pytest.raises(TypeError, match="PagedKVCacheFp8"):
            model(dec, cache).run(torch.ones(1), None)
