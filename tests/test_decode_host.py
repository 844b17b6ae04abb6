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


@pytest.mark.parametrize("call", ["capture", "capture_run"])
def test_capture_records_on_a_stream_of_the_inputs_device(dec, monkeypatch, call):
    """torch's own capture stream belongs to the device that was current when it was made: a model on another one
    would launch outside the capture, and the graph would be empty."""
    from contextlib import contextmanager

    class Stream:
        def __init__(self, device=None):
            self.device = device

        def wait_stream(self, other):
            pass

    current, recorded = [], []

    @contextmanager
    def use(stream):
        current.append(stream)
        yield
        current.pop()

    @contextmanager
    def graph(g, stream=None):
        with use(stream or Stream("another")):
            recorded.append("begin")
            yield
            recorded.append("end")

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", use)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    note = lambda *args, **kw: recorded.append(current[-1].device) or args[0]  # noqa: E731
    m = model(dec, dec.PagedKVCacheFp8(2, 1, 1, "cpu"))
    monkeypatch.setattr(m, "step", note)
    monkeypatch.setattr(m, "plan", note)
    monkeypatch.setattr(m, "run", note)
    x = torch.ones(1)
    _, statics, out, *_ = m.capture(x, x, x, x) if call == "capture" else m.capture_run(x, x, x, x, x, 1)
    assert out is statics[0]
    captured = recorded[recorded.index("begin") + 1:recorded.index("end")]
    assert captured and all(d == x.device for d in captured)
