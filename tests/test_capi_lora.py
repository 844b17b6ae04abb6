"""Adapters and token log probabilities on the CPU: size queries and the checks that return before a launch."""

from __future__ import annotations

import ctypes
import os
from types import SimpleNamespace

import pytest
import torch

FAKE = 0x10000  # 16-byte aligned, never dereferenced on these paths


@pytest.fixture(scope="module")
def lib(pkg):
    from inference_server_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__

        __graft_entry__._load_build_module().build()
    return _lib.load()


def ints(*v):
    return (ctypes.c_int * len(v))(*v)


def test_plan_sizes(lib):
    at = (ctypes.c_int32 * 2)()
    n = lib.moe_mi355x_lora_plan_bytes(100, 7, at)
    offsets, rows = at
    assert 0 < offsets and rows - offsets == 7 + 2 and n >= 4 * (rows + 100)
    for T, L in ((101, 7), (100, 8), (1 << 18, 256)):
        assert lib.moe_mi355x_lora_plan_bytes(T, L, None) >= n
    for T, L in ((-1, 1), ((1 << 18) + 1, 1), (1, 0), (1, 257)):
        assert lib.moe_mi355x_lora_plan_bytes(T, L, None) == 0
    assert lib.moe_mi355x_lora_plan_bytes(0, 1, None) > 0


def test_plan_refusals(lib):
    n = lib.moe_mi355x_lora_plan_bytes(8, 4, None)

    def call(ids=FAKE, cu=FAKE, seqs=2, T=8, L=4, plan=FAKE, size=n):
        return lib.moe_mi355x_lora_plan(ids, cu, seqs, T, L, plan, size, None)

    assert call(T=-1) == -1 and call(L=0) == -1 and call(L=257) == -1 and call(T=(1 << 18) + 1) == -1
    assert call(seqs=-1) == -1 and call(seqs=4097) == -1
    assert call(ids=None) == -1 and call(ids=None, cu=None) == -1
    assert call(plan=None) == -2 and call(size=n - 1) == -2
    assert call(plan=FAKE + 4) == -3


def test_add_workspace(lib):
    """Small steps need none; larger ones hold A x of every row and part, once at least."""
    ws = lib.moe_mi355x_lora_add_workspace_bytes
    assert ws(1, 4, 256, 16, 1, ints(64)) == 0
    assert ws(5000, 4, 2048, 64, 3, ints(4096, 512, 512)) >= 5000 * 3 * 64 * 4
    for bad in ((-1, 4, 256, 16, 1), (1, 0, 256, 16, 1), (1, 4, 40, 16, 1), (1, 4, 256, 8, 1), (1, 4, 256, 144, 1),
                (1, 4, 256, 16, 0), (1, 4, 256, 16, 5)):
        assert ws(*bad, ints(64, 64, 64, 64, 64)) == 0
    assert ws(5000, 4, 256, 16, 1, None) == 0


def test_add_refusals(lib):
    T, L, K, R, columns = 5000, 4, 256, 16, ints(64, 32)
    n = lib.moe_mi355x_lora_add_workspace_bytes(T, L, K, R, 2, columns)
    assert n > 0

    def call(y=FAKE, ys=96, x=FAKE, xs=K, a=FAKE, b=FAKE, ranks=FAKE, scales=FAKE, plan=FAKE, T=T, L=L, K=K, R=R, parts=2,
             columns=columns, ws=FAKE, size=n):
        return lib.moe_mi355x_lora_add(y, ys, x, xs, a, b, ranks, scales, plan, T, L, K, R, parts, columns, ws, size, None)

    for bad in ({"T": -1}, {"L": 0}, {"L": 257}, {"K": 0}, {"K": 250}, {"R": 0}, {"R": 20}, {"R": 144}, {"parts": 0}, {"parts": 5},
                {"columns": None}, {"columns": ints(64, 30)}, {"columns": ints(64, 0)}, {"columns": ints(1 << 24, 32)},
                {"ys": 95}, {"xs": 255}, *({k: None} for k in ("y", "x", "a", "b", "ranks", "scales", "plan"))):
        assert call(**bad) == -1, bad
    for bad in ({"ys": 100}, {"xs": 260}, {"y": FAKE + 2}, {"x": FAKE + 8}, {"a": FAKE + 4}, {"b": FAKE + 2}, {"plan": FAKE + 4},
                {"ws": FAKE + 4}):
        assert call(**bad) == -3, bad
    assert call(ws=None) == -2 and call(size=n - 1) == -2
    assert call(T=0, y=None, x=None, ws=None) == 0  # no rows: nothing to do


def test_logprobs_refusals(lib):
    ws = lib.moe_mi355x_token_logprobs_workspace_bytes
    n = ws(3, 100000, 5)
    assert n > 0 and ws(3, 1000, 5) == 0 and ws(100000, 100000, 5) == 0
    for bad in ((-1, 10, 0), (1 << 24, 10, 0), (1, 0, 0), (1, 10, 11), (1, 100, 65), (1, 100, -1)):
        assert ws(*bad) == 0

    def call(x=FAKE, dtype=0, stride=100000, tokens=FAKE, idb=8, T=3, V=100000, k=5, lp=FAKE, h=FAKE, ids=FAKE, top=FAKE, w=FAKE,
             size=n):
        return lib.moe_mi355x_token_logprobs(x, dtype, stride, tokens, idb, T, V, k, lp, h, ids, top, w, size, None)

    for bad in ({"dtype": 2}, {"stride": 99999}, {"idb": 2}, {"T": -1}, {"T": 1 << 24}, {"V": 0}, {"k": 65}, {"k": -1}, {"x": None},
                {"h": None}, {"lp": None}, {"ids": None}, {"top": None}):
        assert call(**bad) == -1, bad
    assert call(x=FAKE + 1) == -3 and call(dtype=1, x=FAKE + 2) == -3 and call(w=FAKE + 8) == -3
    assert call(w=None) == -2 and call(size=n - 1) == -2
    assert call(T=0, x=None) == 0


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu(pkg):
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        pkg.lora_plan(one, 1)
    with pytest.raises(ValueError, match="GPU"):
        pkg.token_logprobs(torch.zeros((1, 4)))
    with pytest.raises(ValueError, match="GPU"):
        pkg.LoraPool.empty(1, 32, (32,), 16, "cpu")
    with pytest.raises(TypeError, match="LoraPool"):
        pkg.lora_add(one, one, None, None)
    with pytest.raises(TypeError):
        pkg.lora_plan([1], 1)
    with pytest.raises(TypeError):
        pkg.token_logprobs(torch.zeros((1, 4), dtype=torch.float16))


# ---- the decode step's adapters, with stand-ins for pools and kernels ----


@pytest.fixture
def dec(pkg):
    from inference_server_amd import decode

    return decode


def test_models_take_adapters_of_one_number(dec):
    pool = lambda n: SimpleNamespace(num_adapters=n)  # noqa: E731
    layers = [SimpleNamespace(wqkv=torch.zeros(1)) for _ in range(2)]
    make = lambda *a: dec.DecodeModel(dec.DecoderConfig(), layers, dec.PagedKVCache(2, 1, 1, "cpu"), list(a))  # noqa: E731
    A = dec.LayerAdapters
    assert make(A(pool(3), pool(3)), A(None, pool(3))).num_adapters == 3
    for bad in ((A(pool(3)),), (A(pool(3)), A(pool(2))), (A(), A())):
        with pytest.raises(ValueError):
            make(*bad)
    without = dec.DecodeModel(dec.DecoderConfig(), layers, dec.PagedKVCache(2, 1, 1, "cpu"))
    x = torch.ones(1)
    for call in (lambda: without.lora_plan(x), lambda: without.step(x, x, x, x, lora=object()),
                 lambda: without.capture(x, x, x, x, adapter_ids=x)):
        with pytest.raises(ValueError, match="without adapters"):
            call()


def test_projections_add_where_there_is_a_pool_and_a_plan(dec, monkeypatch):
    calls = []
    monkeypatch.setattr(dec, "_linear", lambda x, w: x * w)
    monkeypatch.setattr(dec.kernels, "lora_add", lambda y, x, pool, plan: calls.append((pool, plan)) or y + 1)
    x = torch.ones(2)
    assert dec._project(x, 3.0, None, "plan").tolist() == [3, 3] and dec._project(x, 3.0, "pool", None).tolist() == [3, 3]
    assert not calls and dec._project(x, 3.0, "pool", "plan").tolist() == [4, 4] and calls == [("pool", "plan")]


def test_rows_of_logits_end_at_2_30(lib):
    """A place in a row, and a vector's past its end, stay ints; the split of one row over workgroups too."""
    ws = lib.moe_mi355x_token_logprobs_workspace_bytes
    assert ws(1, 1 << 30, 5) > 0
    for V in ((1 << 30) + 1, (1 << 31) - 4096, (1 << 31) - 1):
        assert ws(1, V, 5) == 0
        assert lib.moe_mi355x_token_logprobs(FAKE, 0, 1 << 32, FAKE, 8, 1, V, 5, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == -1


@pytest.mark.parametrize("at,ys,xs,T", [
    (0, 96, 256, 5000), (64, 96, 256, 5000), (-256, 96, 256, 5000), (5000 * 96 - 8, 96, 256, 5000), (88, 352, 352, 5000),
    (104, 352, 352, 5000), (-248, 352, 352, 5000), (7 * 352, 352, 352, 5000), (88, 352, 352, 1), (-248, 96, 256, 1)])
def test_add_refuses_an_x_that_it_would_change(lib, at, ys, xs, T):
    """x `at` values behind y, K 256 and N 96."""
    y = 1 << 30
    n = lib.moe_mi355x_lora_add_workspace_bytes(T, 4, 256, 16, 2, ints(64, 32))
    assert lib.moe_mi355x_lora_add(y, ys, y + 2 * at, xs, FAKE, FAKE, FAKE, FAKE, FAKE, T, 4, 256, 16, 2, ints(64, 32), FAKE, n,
                                   None) == -1


# ---- loading adapters, over CPU tensors (a pool's own constructor takes GPU tensors alone) ----


def pool_on_cpu(pkg, L, K, columns, R):
    pool = object.__new__(pkg.LoraPool)
    pool.a, pool.b = torch.zeros((L, len(columns) * R, K)), torch.zeros((L, sum(columns), R))
    pool.ranks, pool.scales = torch.zeros(L, dtype=torch.int32), torch.zeros(L)
    pool.columns, pool.in_features, pool.out_features, pool.max_rank, pool.num_adapters = columns, K, sum(columns), R, L
    return pool


def test_trained_weights_are_loaded_as_values(pkg):
    """Parameters that take gradients leave none of their graph in the pool, whose own tensors may take them too."""
    pool = pool_on_cpu(pkg, 2, 32, (32,), 16)
    a, b = (torch.nn.Parameter(torch.randn(s)) for s in ((4, 32), (32, 4)))
    pool.load(0, [(a, b)], 1.0)
    assert not pool.a.requires_grad and not pool.b.requires_grad
    pool.a, pool.b = pool.a.requires_grad_(), pool.b.requires_grad_()
    pool.load(1, [(a, b)], 1.0)
    assert pool.a.is_leaf and pool.b.is_leaf
    for i in range(2):
        assert torch.equal(pool.a[i, :4], a) and torch.equal(pool.b[i, :, :4], b)


def test_an_adapter_is_loaded_from_the_pool_itself(pkg):
    """From its own slot with another scale, its parts changed over, cut to a lower rank; and from another slot."""
    pool = pool_on_cpu(pkg, 2, 32, (32, 32), 16)
    parts = [(torch.randn(4, 32), torch.randn(32, 4)) for _ in range(2)]

    def held(slot, r):
        return [(pool.a[slot, 16 * p:16 * p + r], pool.b[slot, 32 * p:32 * p + 32, :r]) for p in range(2)]

    def check(slot, want):
        for p, (a, b) in enumerate(want):
            r = len(a)
            mine_a, mine_b = pool.a[slot, 16 * p:16 * p + 16], pool.b[slot, 32 * p:32 * p + 32]
            assert torch.equal(mine_a[:r], a) and torch.equal(mine_b[:, :r], b)
            assert not mine_a[r:].any() and not mine_b[:, r:].any()

    pool.load(0, parts, 1.0)
    pool.load(0, held(0, 4), 0.5)
    check(0, parts)
    pool.load(0, held(0, 4)[::-1], 0.5)
    check(0, parts[::-1])
    pool.load(1, held(0, 4), 2.0)
    check(1, parts[::-1])
    pool.load(0, held(0, 3), 1.0)
    check(0, [(a[:3], b[:, :3]) for a, b in parts[::-1]])
    assert pool.ranks.tolist() == [3, 4] and pool.scales.tolist() == [1.0, 2.0]


def test_models_take_pools_of_their_own_projections(pkg, dec):
    """Columns in another order or in other parts, of the same sum, would be added to other columns."""
    cfg = dec.DecoderConfig(hidden=64, heads=2, kv_heads=1)
    q, k, v = dec.LayerAdapters.qkv_columns(cfg)
    layers = [SimpleNamespace(wqkv=torch.zeros(1), cfg=cfg)]

    def pool(K, columns, device=-1):
        p = pool_on_cpu(pkg, 2, K, columns, 16)
        p.device = device
        return p

    def make(qkv=pool(64, (q, k, v)), o=pool(q, (64,))):
        return dec.DecodeModel(cfg, layers, dec.PagedKVCache(1, 1, 1, "cpu"), [dec.LayerAdapters(qkv, o)])

    make(), make(qkv=None), make(o=None)
    for bad in ({"qkv": pool(64, (k, v, q))}, {"qkv": pool(64, (q + k + v,))}, {"qkv": pool(64, (q, k + v))},
                {"qkv": pool(96, (q, k, v))}, {"qkv": pool(64, (q, k, v), device=0)}, {"o": pool(q, (32, 32))}, {"o": pool(64, (q,))},
                {"o": pool(q, (64,), device=1)}):
        with pytest.raises(ValueError, match="qkv|o "):
            make(**bad)
    wrong = dec.LayerAdapters(pool(64, (k, v, q)))
    for sublayer, n in ((dec.attention_sublayer, 6), (dec.attention_sublayer_fp8, 6)):
        with pytest.raises(ValueError, match="qkv"):
            sublayer(layers[0], torch.zeros((1, 64)), *[None] * n, adapters=wrong, lora=object())
