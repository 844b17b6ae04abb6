"""The 8-bit paged KV cache's entry points on the CPU: size queries and the checks that return before a launch."""

from __future__ import annotations

import ctypes
import os

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


def shape(pkg, *sizes):
    return ctypes.byref(pkg._lib.PlanShape(*sizes))


def test_plan_sizes(pkg, lib):
    at = (ctypes.c_int32 * 5)()
    n = lib.moe_mi355x_paged_plan_bytes(shape(pkg, 3, 40, 40, 9, 32, 4), at)
    pages, cu, ctx, pos, slot = at
    assert 0 <= pages < cu and (ctx - cu, pos - ctx, slot - pos) == (4, 3, 40) and 4 * (slot + 40) < n
    # more of anything takes no less
    base = (64, 512, 512, 100, 32, 4)
    size = lib.moe_mi355x_paged_plan_bytes(shape(pkg, *base), None)
    for i, v in ((0, 65), (1, 600), (3, 1000)):
        assert lib.moe_mi355x_paged_plan_bytes(shape(pkg, *base[:i], v, *base[i + 1:]), None) >= size
    assert lib.moe_mi355x_paged_plan_bytes(None, None) == 0
    for bad in [(-1, 1, 1, 1, 4, 4), (4097, 1, 1, 1, 4, 4), (1, -1, 1, 1, 4, 4), (1, (1 << 18) + 1, 1, 1, 4, 4),
                (1, 1, 0, 1, 4, 4), (1, 1, 1, 0, 4, 4), (1, 1, 1, (1 << 22) + 1, 4, 4), (1, 1, 1, 1, 5, 4), (1, 1, 1, 1, 17, 1),
                (1, 1, 1, 1, 0, 1), (1, 1, 1, 1, 4, 0), (1, 1, 1, 1, 2048, 2048)]:
        assert lib.moe_mi355x_paged_plan_bytes(shape(pkg, *bad), None) == 0, bad
        assert lib.moe_mi355x_paged_attn_fp8_workspace_bytes(shape(pkg, *bad)) == 0, bad
    for good in [(0, 0, 1, 1, 1, 1), (4096, 1 << 18, 1 << 18, 1 << 22, 16, 1), (1, 1, 1, 1, 1024, 1024)]:
        assert lib.moe_mi355x_paged_plan_bytes(shape(pkg, *good), None) > 0, good


def test_workspace_only_where_something_can_be_split(pkg, lib):
    ws = lib.moe_mi355x_paged_attn_fp8_workspace_bytes
    assert ws(shape(pkg, 1, 1, 1, 65, 32, 4)) == 0            # a decode step over small tables
    assert ws(shape(pkg, 128, 128, 1, 512, 32, 4)) > 0
    assert ws(shape(pkg, 2, 200, 150, 16, 32, 4)) == 0         # prompts of up to 256 tokens
    assert ws(shape(pkg, 2, 200, 150, 100, 32, 4)) > 0


def test_plan_refusals(pkg, lib):
    good = (2, 4, 4, 8, 32, 4)
    n = lib.moe_mi355x_paged_plan_bytes(shape(pkg, *good), None)
    call = lambda s=good, free=0, plan=FAKE, size=n, cached=FAKE, new=FAKE, tables=FAKE, pages=FAKE: \
        lib.moe_mi355x_paged_plan(cached, new, tables, pages, free, shape(pkg, *s), plan, size, None)  # noqa: E731
    assert call(s=(2, 4, 4, 8, 33, 4)) == -1
    assert call(free=-1) == -1
    assert call(cached=None) == -1 and call(new=None) == -1 and call(tables=None) == -1
    assert call(free=3, pages=None) == -1
    assert call(plan=None) == -2 and call(size=n - 4) == -2
    assert call(plan=FAKE + 4) == -3


def test_append_refusals(pkg, lib):
    good = (2, 4, 4, 8, 32, 4)

    def call(k=FAKE, ks=512, kc=FAKE, s=good, hd=128, ps=16, pages=9, plan=FAKE):
        return lib.moe_mi355x_kv_append_fp8(k, FAKE, ks, 512, kc, FAKE, FAKE, FAKE, hd, ps, pages, shape(pkg, *s), plan, None)

    assert call(hd=64) == -1 and call(ps=32) == -1 and call(pages=-1) == -1 and call(s=(2, 4, 4, 8, 33, 4)) == -1
    assert call(k=None) == -1 and call(kc=None) == -1 and call(plan=None) == -1 and call(ks=500) == -1
    assert call(k=FAKE + 2) == -3 and call(kc=FAKE + 8) == -3 and call(ks=516) == -3
    assert call(k=None, s=(2, 0, 4, 8, 32, 4)) == 0  # no tokens: nothing to do

    def fused(qkv=FAKE, q=FAKE, s=good, hd=128):
        return lib.moe_mi355x_qk_norm_rope_append_fp8(qkv, FAKE, FAKE, FAKE, 1e-6, q, FAKE, FAKE, FAKE, FAKE, hd, 16, 9,
                                                      shape(pkg, *s), FAKE, None)

    assert fused(hd=64) == -1 and fused(qkv=None) == -1 and fused(q=None) == -1
    assert fused(qkv=FAKE + 2) == -3 and fused(q=FAKE + 8) == -3
    assert fused(qkv=None, s=(2, 0, 4, 8, 32, 4)) == 0


def test_attention_refusals(pkg, lib):
    good = (128, 128, 1, 512, 32, 4)
    n = lib.moe_mi355x_paged_attn_fp8_workspace_bytes(shape(pkg, *good))

    def call(q=FAKE, stride=4096, tables=FAKE, s=good, scale=0.1, hd=128, ps=16, pages=9, out=FAKE, ws=FAKE, size=n):
        return lib.moe_mi355x_paged_attn_fp8(q, stride, FAKE, FAKE, FAKE, FAKE, tables, hd, ps, pages, scale, shape(pkg, *s),
                                             FAKE, out, ws, size, None)

    assert call(hd=64) == -1 and call(ps=32) == -1 and call(pages=-1) == -1 and call(s=(128, 128, 1, 512, 33, 4)) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == -1
    assert call(q=None) == -1 and call(tables=None) == -1 and call(out=None) == -1 and call(stride=4000) == -1
    assert call(q=FAKE + 2) == -3 and call(out=FAKE + 8) == -3 and call(stride=4100) == -3
    assert call(ws=None) == -2 and call(size=n - 1) == -2
    assert call(q=None, s=(2, 0, 4, 8, 32, 4)) == 0


def test_wrappers_refuse_tensors_that_are_not_on_a_gpu(pkg):
    one, tables = torch.ones(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        pkg.paged_plan(one, one, tables, one, 1, 1, 32, 4)
    with pytest.raises(TypeError):
        pkg.paged_plan(one, one, None, one, 1, 1, 32, 4)
    for call in (lambda p: pkg.kv_append_fp8(one, one, one, one, one, one, p),
                 lambda p: pkg.paged_attention_fp8(one, one, one, one, one, p, 0.1)):
        with pytest.raises(TypeError, match="PagedPlan"):
            call(None)


def test_unpack_tells_the_pools_apart(pkg):
    k = torch.zeros((2, 1, 8, 16, 16), dtype=torch.float8_e4m3fn)
    v = torch.zeros((2, 1, 2, 4, 64, 4), dtype=torch.float8_e4m3fn)
    s = torch.full((2, 1), 0.5)
    k[1, 0, 3, 5, 7] = 4.0   # token 5, dim 55
    v[1, 0, 1, 2, 9, 3] = 4.0  # token 11, dim 73
    a, b = pkg.unpack_kv_fp8(k, s), pkg.unpack_kv_fp8(v, s)
    assert a.shape == b.shape == (2, 1, 16, 128)
    assert a[1, 0, 5, 55] == 2.0 and b[1, 0, 11, 73] == 2.0 and a.sum() == b.sum() == 2.0
    with pytest.raises(ValueError):
        pkg.unpack_kv_fp8(k, s[:1])
    with pytest.raises(ValueError):
        pkg.unpack_kv_fp8(k.float(), s)


def test_attention_refuses_a_scale_past_fp32(pkg, lib):
    """The kernels work with scale * log2(e): infinite, it would make NaN of a score of 0."""
    good = (128, 128, 1, 512, 32, 4)
    n = lib.moe_mi355x_paged_attn_fp8_workspace_bytes(shape(pkg, *good))

    def call(scale, ws):
        return lib.moe_mi355x_paged_attn_fp8(FAKE, 4096, FAKE, FAKE, FAKE, FAKE, FAKE, 128, 16, 9, scale, shape(pkg, *good),
                                             FAKE, FAKE, ws, n, None)

    for scale in (2.4e38, 3.4e38):
        assert call(scale, None) == -1
    for scale in (2.3e38, 1e-38):  # taken, so the next check answers
        assert call(scale, None) == -2
