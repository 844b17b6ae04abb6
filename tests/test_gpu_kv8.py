"""The 8-bit paged KV cache on the GPU (plan, quantising writers, attention) against oracle/kv8_oracle.py, in 64 bits.

Tolerances, from the roundings alone.  A bf16 value is off by half a step, 2^-8 of it; an e4m3 code by 2^-4 of its
value or, among the subnormals, 2^-10 scales.
  attention: with p the probabilities, each rounded to bf16 for the product with V, p' = p (1 + d), |d| <= 2^-8, and
    the tiles' sum formed from the rounded ones, o' = sum p' v / sum p' differs from o = sum p v (sum p = 1) by
    |sum p d (v - o)| / |sum p'| <= 2^-8 (sum p |v| + |o|) (1 + 2^-8); rounding the result adds 2^-8 |o|.  5% more
    covers the (1 + 2^-8) and the fp32 scores: 128 products summed in fp32 are off by 128 * 2^-24 of their sum of
    |q k| at most, with scale sum |q k| below 25 here 2e-4 of each p, which is 5% of 2^-8.
  norm and rotary: r, the weight, the angle (rounded to 2^-25 of a turn: 2^-22 radians), cos, sin and the two
    products in fp32 are each off by a few 2^-24: 2^-19 of |a| + |b| in all, beside the one rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8_oracle as kv
from oracle import moe_oracle as orc
from tests.helpers import to_bf16

pytestmark = pytest.mark.gpu

PAGE, D = 16, 128
SCALE = D ** -0.5
FP8 = torch.float8_e4m3fn
K_SHAPE, V_SHAPE = (8, 16, 16), (2, 4, 64, 4)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(dev)


class Step:
    """A step on a cache in use: tables of the cached tokens, free pages, pools of random codes and scales."""

    def __init__(self, pkg, dev, cached, new, Hq, Hkv, seed=0, T=None, max_new=None, spare=3, width=None, free=None,
                 poison=False):
        rng = self.rng = np.random.default_rng(seed)
        self.pkg, self.dev, self.Hq, self.Hkv = pkg, dev, Hq, Hkv
        self.cached, self.new = list(cached), list(new)
        B = len(self.cached)
        self.T = sum(self.new) if T is None else T
        self.max_new = max([1, *self.new]) if max_new is None else max_new
        have = [-(-c // PAGE) for c in self.cached]
        want = [-(-(c + n) // PAGE) for c, n in zip(self.cached, self.new)]
        self.pages = sum(want) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.width = max([1, *want]) + 2 if width is None else width
        self.tables = np.full((B, self.width), -1, np.int32)
        at = 0
        for b in range(B):
            n = min(have[b], self.width)
            self.tables[b, :n] = order[at:at + n]
            at += have[b]
        self.free = order[at:] if free is None else np.asarray(free, np.int32)
        self.k = rng.integers(0, 256, (self.pages, Hkv, *K_SHAPE)).astype(np.uint8)
        self.v = rng.integers(0, 256, (self.pages, Hkv, *V_SHAPE)).astype(np.uint8)
        if not poison:  # NaN codes become zeros
            self.k[(self.k & 127) == 127] = 0
            self.v[(self.v & 127) == 127] = 0
        self.ks = (2.0 ** rng.integers(-9, -6, (self.pages, Hkv))).astype(np.float32)
        self.vs = (2.0 ** rng.integers(-9, -6, (self.pages, Hkv))).astype(np.float32)
        self.ref = kv.plan(self.cached, self.new, self.tables, self.free, self.T, self.max_new)
        self.g_tables, self.g_free = i32(self.tables, dev), i32(self.free, dev)
        self.g_cached, self.g_new = i32(self.cached, dev), i32(self.new, dev)
        self.cache = tuple(torch.from_numpy(x).to(dev) for x in (self.k, self.v, self.ks, self.vs))
        self.cache = (self.cache[0].view(FP8), self.cache[1].view(FP8), *self.cache[2:])

    def plan(self, out=None):
        return self.pkg.paged_plan(self.g_cached, self.g_new, self.g_tables, self.g_free, self.T, self.max_new, self.Hq,
                                   self.Hkv, out=out)

    def got(self):
        """The cache as the GPU has it."""
        torch.cuda.synchronize()
        k, v, ks, vs = self.cache
        return k.view(torch.uint8).cpu().numpy(), v.view(torch.uint8).cpu().numpy(), ks.cpu().numpy(), vs.cpu().numpy()

    def check_plan(self, p):
        pos, slot, cu, ctx, tables, used = self.ref
        torch.cuda.synchronize()
        assert np.array_equal(p.positions.cpu().numpy(), pos)
        assert np.array_equal(p.slots.cpu().numpy(), slot)
        assert np.array_equal(p.cu_tokens.cpu().numpy(), cu)
        assert np.array_equal(p.context_lens.cpu().numpy(), ctx)
        assert np.array_equal(p.block_tables.cpu().numpy(), tables)
        assert p.pages_used.item() == used

    def attention_ref(self, q):
        k, v, ks, vs = self.got()
        return kv.attention(q, kv.unpack(k, ks, kv.k_index), kv.unpack(v, vs, kv.v_index), self.ref[2], self.ref[0],
                            self.ref[4], SCALE)

    def check_attention(self, p, q_std=1.0):
        q = orc.round_bf16((self.rng.standard_normal((self.T, self.Hq, D)) * q_std).astype(np.float32))
        o = self.pkg.paged_attention_fp8(to_bf16(q, self.dev), *self.cache, p, SCALE)
        assert o.shape == (self.T, self.Hq, D) and o.dtype == torch.bfloat16
        self.check_output(o, q)

    def check_output(self, o, q):
        ref, size = self.attention_ref(q)
        got = o.float().cpu().numpy()
        assert np.isfinite(got).all()
        worst = np.abs(got - ref) - 2.0 ** -8 * (1.05 * (size + np.abs(ref)) + np.abs(ref))
        assert (worst <= 1e-30).all(), (worst.max(), np.argwhere(worst > 0)[:4])


# lengths: one token, page edges, odd ones, empty sequences among them
LENS = [
    ([0], [1]),
    ([0, 15, 16, 17, 31], [1, 1, 1, 1, 1]),
    ([5, 0, 0, 300, 47], [0, 17, 0, 1, 33]),
    ([0, 100, 1000, 16], [130, 64, 1, 500]),
]


@pytest.mark.parametrize("cached,new", LENS)
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (7, 7)])
def test_plan_matches_oracle(pkg, dev, cached, new, Hq, Hkv):
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=1)
    s.check_plan(s.plan())


@pytest.mark.parametrize("B", [1024, 1025, 4096])
def test_plan_many_sequences(pkg, dev, B):
    rng = np.random.default_rng(B)
    new = rng.integers(0, 3, B)
    new[rng.integers(0, B, 5)] = 200
    s = Step(pkg, dev, rng.integers(0, 200, B), [int(n) for n in new], 32, 4, seed=2)
    s.check_plan(s.plan())


def test_plan_padding_overflow_and_bad_lengths(pkg, dev):
    """Rows behind the last sequence; more tokens than rows; more than max_new; more than the table holds; more pages than
    are free; lengths below zero and past the table."""
    s = Step(pkg, dev, [3, 40], [5, 20], 32, 4, T=64)
    s.check_plan(s.plan())
    s = Step(pkg, dev, [3, 40, 7], [5, 20, 9], 32, 4, T=17)
    s.check_plan(s.plan())
    s = Step(pkg, dev, [3, 40, 7], [5, 20, 9], 32, 4, max_new=6, T=15)
    s.check_plan(s.plan())
    s = Step(pkg, dev, [10, 70], [60, 1], 32, 4, width=3)
    s.check_plan(s.plan())
    s = Step(pkg, dev, [10, 30], [60, 70], 32, 4, free=[1, 0])
    s.check_plan(s.plan())
    s = Step(pkg, dev, [0, 20], [4, 4], 32, 4, T=8)
    s.cached, s.new = [-5, 1 << 30], [-3, 4]
    s.g_cached, s.g_new = i32(s.cached, dev), i32(s.new, dev)
    s.ref = kv.plan(s.cached, s.new, s.tables, s.free, s.T, s.max_new)
    s.check_plan(s.plan())


def test_plan_without_tokens_or_sequences(pkg, dev):
    s = Step(pkg, dev, [3, 16], [0, 0], 32, 4)
    p = s.plan()
    s.check_plan(p)
    s.check_attention(p)
    s = Step(pkg, dev, [], [], 32, 4, T=5)
    p = s.plan()
    assert p.cu_tokens.tolist() == [0] and p.positions.tolist() == [-1] * 5 and p.pages_used.item() == 0
    s.check_attention(p)
    before = s.got()
    x = torch.ones((5, 4, D), dtype=torch.bfloat16, device=dev)
    pkg.kv_append_fp8(x, x, *s.cache, p)
    q = pkg.qk_norm_rope_append_fp8(torch.ones((5, 40 * D), dtype=torch.bfloat16, device=dev), x[0, 0], x[0, 0],
                                    torch.ones(64, device=dev), 32, 4, 1e-6, *s.cache, p)
    assert (q == 0).all() and all(np.array_equal(a, b) for a, b in zip(before, s.got()))
    s = Step(pkg, dev, [3, 16], [0, 0], 32, 4, T=0)
    p = s.plan()
    s.check_plan(p)
    pkg.kv_append_fp8(x[:0], x[:0], *s.cache, p)
    assert pkg.paged_attention_fp8(x[:0].reshape(0, 1, 4, D).expand(0, 8, 4, D).reshape(0, 32, D), *s.cache, p, SCALE).shape == \
        (0, 32, D)


def new_kv(s, outliers=True):
    k = s.rng.standard_normal((s.T, s.Hkv, D)) * (np.exp2(np.abs(s.rng.standard_normal((s.Hkv, D)))) if outliers else 1)
    return orc.round_bf16(k.astype(np.float32)), orc.round_bf16(s.rng.standard_normal((s.T, s.Hkv, D)).astype(np.float32))


def check_append(s, k, v):
    ek, ev, eks, evs = s.k.copy(), s.v.copy(), s.ks.copy(), s.vs.copy()
    kv.append(k, s.ref[1], s.ref[0], ek, eks, kv.k_index)
    kv.append(v, s.ref[1], s.ref[0], ev, evs, kv.v_index)
    gk, gv, gks, gvs = s.got()
    assert np.array_equal(gks, eks) and np.array_equal(gvs, evs)
    # a code's NaN has no sign to speak of
    nan = lambda c: np.where((c & 127) == 127, 127, c)  # noqa: E731
    assert np.array_equal(nan(gk), nan(ek)) and np.array_equal(nan(gv), nan(ev))


@pytest.mark.parametrize("cached,new", LENS)
@pytest.mark.parametrize("Hkv", [1, 4, 7])
def test_append_matches_oracle(pkg, dev, cached, new, Hkv):
    s = Step(pkg, dev, cached, new, Hkv, Hkv, seed=3)
    k, v = new_kv(s)
    pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *s.cache, s.plan())
    check_append(s, k, v)


def test_append_token_by_token_grows_the_scale(pkg, dev):
    """A page filled one token at a time, each larger than the last: the scale grows and the codes are re-coded."""
    s = Step(pkg, dev, [0, 5], [1, 1], 4, 4, seed=4)
    k0, v0 = new_kv(s)
    seen = []
    for step in range(20):
        s.cached, s.new = [step, 5 + step], [1, 1]
        s.g_cached = i32(s.cached, dev)
        s.tables = s.ref[4]
        s.free = s.free[s.ref[5]:] if step else s.free
        s.g_free = i32(s.free, dev)
        s.k, s.v, s.ks, s.vs = s.got()
        s.ref = kv.plan(s.cached, s.new, s.tables, s.free, s.T, 1)
        k, v = orc.round_bf16(k0 * np.float32(1.5 ** step)), orc.round_bf16(v0 * np.float32(0.7 ** step))
        pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *s.cache, s.plan())
        check_append(s, k, v)
        seen.append(s.got()[2].max())
    assert len(set(seen)) > 5


def test_append_special_values(pkg, dev):
    """Zeros, the smallest and largest bf16 values, infinities and NaN: no scale from a non-finite value."""
    s = Step(pkg, dev, [0, 9], [16, 5], 2, 2, seed=5)
    k, v = new_kv(s)
    k[0], v[1] = 0, 0
    k[2, 0, 3], k[3, 1, 4], v[4, 0, 7] = np.inf, np.nan, -np.inf
    v[5] = 2.0 ** -133
    k[6, 1] = 3.3e38
    v[17] = 0
    k, v = orc.round_bf16(k), orc.round_bf16(v)
    k[2, 0, 3], k[3, 1, 4], v[4, 0, 7] = np.inf, np.nan, -np.inf
    pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *s.cache, s.plan())
    check_append(s, k, v)
    s = Step(pkg, dev, [0], [3], 2, 2, seed=6)
    z = np.zeros((3, 2, D), np.float32)
    pkg.kv_append_fp8(to_bf16(z, dev), to_bf16(z, dev), *s.cache, s.plan())
    check_append(s, z, z)


def test_append_takes_slices_and_drops_tokens_without_a_page(pkg, dev):
    s = Step(pkg, dev, [10, 30], [60, 70], 32, 4, free=[1, 0, 10 ** 6, -4], T=150)
    k, v = new_kv(s)
    qkv = torch.zeros((s.T, 40, D), dtype=torch.bfloat16, device=dev)
    qkv[:, 32:36], qkv[:, 36:] = to_bf16(k, dev), to_bf16(v, dev)
    pkg.kv_append_fp8(qkv[:, 32:36], qkv[:, 36:], *s.cache, s.plan())
    check_append(s, k, v)


@pytest.mark.parametrize("cached,new", [*LENS, ([100000, 131000], [3, 1])])
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (14, 2), (5, 5)])
def test_qk_norm_rope_append_matches_oracle(pkg, dev, cached, new, Hq, Hkv):
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=7, T=sum(new) + 2)
    x = orc.round_bf16(s.rng.standard_normal((s.T, Hq + 2 * Hkv, D)).astype(np.float32))
    qw, kw = (orc.round_bf16((1 + 0.3 * s.rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    inv_freq = (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    q = pkg.qk_norm_rope_append_fp8(to_bf16(x.reshape(s.T, -1), dev), to_bf16(qw, dev), to_bf16(kw, dev),
                                    torch.from_numpy(inv_freq).to(dev), Hq, Hkv, 1e-6, *s.cache, s.plan())
    pos, slots = s.ref[0], s.ref[1]
    ref, size = kv.norm_rope(x[:, :Hq], qw, inv_freq, pos, 1e-6)
    live = pos >= 0
    got = q.float().cpu().numpy()
    assert (got[~live] == 0).all()
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -19 * size)[live].all()

    k, size = kv.norm_rope(x[:, Hq:Hq + Hkv], kw, inv_freq, pos, 1e-6)
    gk, gv, gks, gvs = s.got()
    ev, evs = s.v.copy(), s.vs.copy()
    kv.append(x[:, Hq + Hkv:], slots, pos, ev, evs, kv.v_index)
    assert np.array_equal(gv, ev) and np.array_equal(gvs, evs)  # v is bf16 already: to the bit
    rows = kv.unpack(gk, gks, kv.k_index)
    for t in np.nonzero(slots >= 0)[0]:
        page, slot = slots[t] // PAGE, slots[t] % PAGE
        scale = gks[page][:, None]
        assert (np.abs(rows[page, :, slot] - k[t]) <= 2.0 ** -4 * np.abs(k[t]) + 2.0 ** -10 * scale + 2.0 ** -18 * size[t]).all()
    ek, eks = s.k.copy(), s.ks.copy()
    kv.append(k, slots, pos, ek, eks, kv.k_index)
    # the scale: the exact one, or its neighbour where the largest key lies within fp32's error of the border
    assert ((gks == eks) | (np.abs(np.log2(gks / eks)) == 1)).all() and (gks != eks).mean() < 0.02


def test_qk_norm_rope_append_codes_are_those_of_64_bits(pkg, dev):
    """Scales and codes of 3 million keys to the bit: the 64-bit forms differ by 1e-12 of a value, and a code's tie lies
    that near for one value in 10^10.  (In fp32 a tie lies within the error for one in 10^6.)"""
    s = Step(pkg, dev, [0, 70000, 21], [3500, 2000, 900], 8, 4, seed=31)
    x = orc.round_bf16(s.rng.standard_normal((s.T, 16, D)).astype(np.float32))
    qw, kw = (orc.round_bf16((1 + 0.3 * s.rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    inv_freq = (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    pkg.qk_norm_rope_append_fp8(to_bf16(x.reshape(s.T, -1), dev), to_bf16(qw, dev), to_bf16(kw, dev),
                                torch.from_numpy(inv_freq).to(dev), 8, 4, 1e-6, *s.cache, s.plan())
    k, _ = kv.norm_rope(x[:, 8:12], kw, inv_freq, s.ref[0], float(np.float32(1e-6)))
    ek, eks = s.k.copy(), s.ks.copy()
    kv.append(k, s.ref[1], s.ref[0], ek, eks, kv.k_index)
    gk, _, gks, _ = s.got()
    assert np.array_equal(gks, eks)
    assert np.array_equal(gk, ek), int((gk != ek).sum())


ATTENTION = [
    ([0], [1]),
    ([0, 15, 16, 17, 31], [1, 1, 1, 1, 1]),           # single tokens around a page's edges
    ([300, 511, 1000, 2047, 63, 0], [1] * 6),         # several steps of a workgroup, one token of context
    ([8191, 5], [1, 1]),                              # split over many workgroups
    ([0], [130]),                                     # a prompt: tiles that are part full
    ([0, 700, 33], [64, 65, 1]),                      # a prompt, a chunk behind cached tokens, a single token
    ([0, 0, 40, 7], [3, 0, 2, 17]),                   # few new tokens, none
    ([3000], [40]),                                   # few tiles: their keys are split
]


@pytest.mark.parametrize("cached,new", ATTENTION)
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (16, 1), (6, 2), (7, 7), (14, 2)])
def test_attention_matches_oracle(pkg, dev, cached, new, Hq, Hkv):
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=sum(cached) + sum(new))
    s.check_attention(s.plan())


def test_attention_long_prompt_and_peaked_scores(pkg, dev):
    s = Step(pkg, dev, [0, 500], [700, 300], 8, 2, seed=11)
    s.check_attention(s.plan(), q_std=8.0)
    s = Step(pkg, dev, [2000, 900], [1, 1], 8, 2, seed=12)
    s.check_attention(s.plan(), q_std=8.0)


def test_attention_ignores_what_lies_behind_a_sequence(pkg, dev):
    """NaN codes in slots behind the last token (their pages end inside a tile) reach no result."""
    s = Step(pkg, dev, [20, 100, 0], [1, 30, 77], 32, 4, seed=13, poison=True, T=115)
    seen = np.zeros((s.pages, PAGE), bool)
    for b in range(3):
        for t in range(s.ref[3][b]):
            seen[s.ref[4][b, t // PAGE], t % PAGE] = True
    pages, slots = np.nonzero(seen)
    d = np.arange(D)
    for codes, index in ((s.k, kv.k_index), (s.v, kv.v_index)):
        for page, slot in zip(pages, slots):
            at = (page, slice(None), *index(slot, d))
            c = codes[at]
            codes[at] = np.where((c & 127) == 127, 0, c)
    s.cache = (torch.from_numpy(s.k).to(dev).view(FP8), torch.from_numpy(s.v).to(dev).view(FP8), *s.cache[2:])
    s.check_attention(s.plan())


def test_attention_leaves_out_pages_that_the_table_does_not_hold(pkg, dev):
    """Stale ids and pads in the middle, a whole prefix without pages, a sequence with none at all."""
    s = Step(pkg, dev, [400, 90, 64, 200], [1, 40, 1, 1], 32, 4, seed=14)
    s.tables[0, 3], s.tables[0, 7:9], s.tables[1, 0], s.tables[2, :4] = -1, 10 ** 6, -5, -1
    s.tables[3, :12] = -1
    s.ref = kv.plan(s.cached, s.new, s.tables, np.full(99, -1), s.T, s.max_new)
    s.g_tables, s.g_free = i32(s.tables, dev), i32(np.full(99, -1), dev)
    s.check_attention(s.plan())


def test_attention_strided_queries_and_other_stream(pkg, dev):
    s = Step(pkg, dev, [50, 0], [1, 90], 32, 4, seed=15)
    q = orc.round_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32))
    wide = torch.zeros((s.T, 40, D), dtype=torch.bfloat16, device=dev)
    wide[:, 8:] = to_bf16(q, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = pkg.paged_attention_fp8(wide[:, 8:], *s.cache, s.plan(), SCALE)
    torch.cuda.current_stream().wait_stream(side)
    s.check_output(o, q)


def test_attention_is_deterministic(pkg, dev):
    s = Step(pkg, dev, [9000, 300, 2000], [1, 1, 60], 32, 4, seed=16)
    p = s.plan()
    q = to_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32), dev)
    a = pkg.paged_attention_fp8(q, *s.cache, p, SCALE)
    for _ in range(3):
        assert torch.equal(a, pkg.paged_attention_fp8(q, *s.cache, p, SCALE))


def test_steps_as_a_server_runs_them(pkg, dev):
    """Prompts, then chunked prefill with decoding sequences, then decode steps, the whole step captured into a graph and
    replayed on lengths that change on the GPU: every step against the oracle's cache and attention."""
    Hq, Hkv, B, T = 32, 4, 3, 48
    s = Step(pkg, dev, [0, 0, 0], [20, 0, 28], Hq, Hkv, seed=17, T=T, max_new=40, spare=24, width=12)
    qkv = torch.zeros((T, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device=dev)
    weight = torch.ones(D, dtype=torch.bfloat16, device=dev)
    inv_freq = torch.from_numpy((1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)).to(dev)
    free, tables = s.free.copy(), s.tables.copy()
    held = {}

    def step():
        held["plan"] = s.plan()
        held["q"] = pkg.qk_norm_rope_append_fp8(qkv.view(T, -1), weight, weight, inv_freq, Hq, Hkv, 1e-6, *s.cache,
                                                held["plan"])
        held["o"] = pkg.paged_attention_fp8(held["q"], *s.cache, held["plan"], SCALE)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s.g_new.zero_()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    cached = [0, 0, 0]
    for new in ([20, 0, 28], [1, 40, 1], [1, 1, 1], [0, 1, 30], [1, 1, 1]):
        s.cached, s.new, s.tables, s.free = list(cached), new, tables, free
        s.ref = kv.plan(cached, new, tables, free, T, s.max_new)
        s.g_cached.copy_(i32(cached, dev))
        s.g_new.copy_(i32(new, dev))
        s.g_free[:len(free)].copy_(i32(free, dev))
        x = orc.round_bf16(s.rng.standard_normal((T, Hq + 2 * Hkv, D)).astype(np.float32))
        qkv.copy_(to_bf16(x, dev))
        s.k, s.v, s.ks, s.vs = s.got()
        graph.replay()
        torch.cuda.synchronize()
        s.check_plan(held["plan"])
        ev, evs = s.v.copy(), s.vs.copy()
        kv.append(x[:, Hq + Hkv:], s.ref[1], s.ref[0], ev, evs, kv.v_index)
        assert np.array_equal(s.got()[1], ev) and np.array_equal(s.got()[3], evs)
        s.check_output(held["o"], held["q"].float().cpu().numpy())
        total = s.ref[2][-1]
        assert (held["o"][total:] == 0).all()
        # the same step eagerly, on the same cache: the same bits
        again = pkg.paged_attention_fp8(held["q"], *s.cache, held["plan"], SCALE)
        assert torch.equal(again, held["o"])
        cached = [c + int(n) for c, n in zip(cached, np.diff(s.ref[2]))]
        tables, free = s.ref[4], free[s.ref[5]:]


def test_refusals(pkg, dev):
    s = Step(pkg, dev, [3, 20], [2, 1], 32, 4)
    p = s.plan()
    k, v, ks, vs = s.cache
    x = torch.zeros((3, 4, D), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((3, 32, D), dtype=torch.bfloat16, device=dev)
    a = (s.g_cached, s.g_new, s.g_tables, s.g_free)
    for bad in [(*a, 3, 2, 32, 5), (*a, 3, 2, 68, 4), (*a, 3, 0, 32, 4), (*a, -1, 2, 32, 4), (*a, (1 << 18) + 1, 2, 32, 4),
                (s.g_cached[:1], *a[1:], 3, 2, 32, 4), (a[0], a[1], a[2][:, 1:], a[3], 3, 2, 32, 4)]:
        with pytest.raises(ValueError):
            pkg.paged_plan(*bad)
    with pytest.raises(TypeError):
        pkg.paged_plan(s.g_cached.long(), *a[1:], 3, 2, 32, 4)
    with pytest.raises(ValueError):
        pkg.paged_plan(*a, 4, 2, 32, 4, out=p)
    for bad in [(x[:2], x, k, v, ks, vs, p), (x, x[:, :2], k, v, ks, vs, p), (x, x, v, k, ks, vs, p), (x, x, k, v[1:], ks, vs, p),
                (x, x, k, v, ks[1:], vs, p), (x, x.transpose(0, 1).contiguous().transpose(0, 1), k, v, ks, vs, p)]:
        with pytest.raises(ValueError):
            pkg.kv_append_fp8(*bad)
    with pytest.raises(TypeError):
        pkg.kv_append_fp8(x.float(), x, k, v, ks, vs, p)
    with pytest.raises(TypeError):
        pkg.kv_append_fp8(x, x, k, v, ks, vs, None)
    with pytest.raises(TypeError):
        pkg.paged_attention_fp8(q, k.view(torch.uint8), v, ks, vs, p, SCALE)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            pkg.paged_attention_fp8(q, k, v, ks, vs, p, scale)
    with pytest.raises(ValueError):
        pkg.paged_attention_fp8(q[:, :16], k, v, ks, vs, p, SCALE)
    off = torch.zeros(3 * 32 * D + 4, dtype=torch.bfloat16, device=dev)[4:].view(3, 32, D)
    with pytest.raises(pkg._lib.MoEKernelError):
        pkg.paged_attention_fp8(off, k, v, ks, vs, p, SCALE)
    with pytest.raises(ValueError):
        pkg.qk_norm_rope_append_fp8(torch.zeros((3, 40 * D), dtype=torch.bfloat16, device=dev), x[0, 0], x[0, 0],
                                    torch.zeros(64, device=dev), 16, 4, 1e-6, k, v, ks, vs, p)


def test_plan_at_its_limits(pkg, dev):
    """2^18 rows: one prompt of them all, and 4096 sequences of 64."""
    s = Step(pkg, dev, [5], [1 << 18], 16, 1, seed=20)
    s.check_plan(s.plan())
    s = Step(pkg, dev, [3] * 4096, [64] * 4096, 16, 1, seed=21)
    s.check_plan(s.plan())


def test_blocks_past_32_bits(pkg, dev):
    """Pools of over 2^32 bytes: pages at both ends, written and read."""
    Hkv, pages = 4, (1 << 32) // (4 * 2048) + 40
    s = Step(pkg, dev, [40, 0, 700], [1, 70, 1], 32, Hkv, seed=22)
    used = s.ref[4][s.ref[4] >= 0]
    high = {int(p): (pages - 1 - i if i % 2 else i) for i, p in enumerate(sorted(set(used.tolist()) | set(s.free.tolist())))}
    big = [torch.zeros((pages, Hkv, *shape), dtype=torch.uint8, device=dev) for shape in (K_SHAPE, V_SHAPE)]
    scales = [torch.ones((pages, Hkv), device=dev) for _ in range(2)]
    for p, q in high.items():
        for dst, src in zip((*big, *scales), (s.k, s.v, s.ks, s.vs)):
            dst[q] = torch.from_numpy(src[p]).to(dev) if src.ndim > 2 else torch.from_numpy(src[p]).to(dev)
    move = lambda a: np.array([high.get(int(x), -1) for x in a.flat], np.int32).reshape(a.shape)  # noqa: E731
    s.g_tables, s.g_free = i32(move(s.tables), dev), i32(move(s.free), dev)
    p = s.plan()
    cache = (big[0].view(FP8), big[1].view(FP8), *scales)
    k, v = new_kv(s)
    pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *cache, p)
    q = orc.round_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32))
    o = pkg.paged_attention_fp8(to_bf16(q, dev), *cache, p, SCALE)
    # the same step on the small pools
    small = Step(pkg, dev, [40, 0, 700], [1, 70, 1], 32, Hkv, seed=22)
    ps = small.plan()
    pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *small.cache, ps)
    assert torch.equal(o, pkg.paged_attention_fp8(to_bf16(q, dev), *small.cache, ps, SCALE))
    small.check_output(o, q)


def test_calls_on_two_streams_share_nothing(pkg, dev):
    """Two attentions of one plan at once, each split over many workgroups, on streams of their own."""
    s = Step(pkg, dev, [9000, 8000], [1, 1], 32, 4, seed=23)
    p = s.plan()
    qs = [to_bf16(s.rng.standard_normal((2, 32, D)).astype(np.float32), dev) for _ in range(2)]
    want = [pkg.paged_attention_fp8(q, *s.cache, p, SCALE) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st, q in zip(streams, qs):
            with torch.cuda.stream(st):
                got.append(pkg.paged_attention_fp8(q, *s.cache, p, SCALE))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(got))


def test_two_graphs_share_nothing(pkg, dev):
    """Attentions of two plans captured into two graphs of one pool, replayed in turn with eager work between."""
    steps = [Step(pkg, dev, [6000, 300], [1, 40], 32, 4, seed=24), Step(pkg, dev, [100, 9000], [50, 1], 32, 4, seed=25)]
    graphs, outs, want = [], [], []
    for s in steps:
        p = s.plan()
        q = to_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32), dev)
        want.append(pkg.paged_attention_fp8(q, *s.cache, p, SCALE))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.paged_attention_fp8(q, *s.cache, p, SCALE))
        graphs.append((g, p, q))
    for _ in range(3):
        for (g, _, _), o, w in zip(graphs, outs, want):
            o.zero_()
            g.replay()
            torch.randn((512, 512), device=dev).sum()
            torch.cuda.synchronize()
            assert torch.equal(o, w)


@pytest.mark.parametrize("T,Hq,Hkv", [(2100, 64, 4), (9000, 16, 1)])
def test_attention_large_tiles(pkg, dev, T, Hq, Hkv):
    """Enough rows for the tiles of 256 of them: every row against a few, computed apart, in 64 bits."""
    s = Step(pkg, dev, [0, 77, 1000], [T - 301, 300, 1], Hq, Hkv, seed=26)
    p = s.plan()
    q = orc.round_bf16(s.rng.standard_normal((T, Hq, D)).astype(np.float32))
    o = pkg.paged_attention_fp8(to_bf16(q, dev), *s.cache, p, SCALE).float().cpu().numpy()
    assert np.isfinite(o).all()
    k, v, ks, vs = s.got()
    k, v = kv.unpack(k, ks, kv.k_index), kv.unpack(v, vs, kv.v_index)
    cu, pos = s.ref[2], s.ref[0]
    some = sorted({0, 1, 15, 16, 17, 63, 64, T - 302, T - 301, T - 2, T - 1, *s.rng.integers(0, T, 25).tolist()})
    for t in some:
        b = int(np.searchsorted(cu, t, side="right")) - 1
        ref, size = kv.attention(q[t:t + 1], k, v, [0, 1], pos[t:t + 1], s.ref[4][b:b + 1], SCALE)
        worst = np.abs(o[t] - ref[0]) - 2.0 ** -8 * (1.05 * (size[0] + np.abs(ref[0])) + np.abs(ref[0]))
        assert (worst <= 1e-30).all(), (t, worst.max())


def check_but(o, ref, size, lost):
    """``o`` is not finite where ``lost`` says so (broadcast to [T, Hq, 128]) and within the module's tolerance elsewhere."""
    got, lost = o.float().cpu().numpy(), np.broadcast_to(lost, o.shape)
    assert not np.isfinite(got[lost]).any(), np.argwhere(np.isfinite(got) & lost)[:4]
    worst = np.abs(got - ref) - 2.0 ** -8 * (1.05 * (size + np.abs(ref)) + np.abs(ref))
    assert (worst[~lost] <= 1e-30).all(), np.argwhere(~(worst <= 1e-30) & ~lost)[:4]


@pytest.mark.parametrize("cached,new", [
    ([300], [1]),                # whole
    ([2000] * 16, [1] * 16),     # split over 8 items
    ([8191], [1]),               # over 64
    ([0], [130]),                # tiles, whole
    ([3000], [40]),              # tiles, split
])
def test_attention_nan_query_gives_nan_whatever_the_split(pkg, dev, cached, new):
    s = Step(pkg, dev, cached, new, 32, 4, seed=40)
    q = orc.round_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32))
    ref, size = s.attention_ref(q)
    lost = np.zeros((s.T, 32, 1), bool)
    lost[s.T // 2, 5] = lost[-1, 31] = True
    o = pkg.paged_attention_fp8(to_bf16(np.where(lost, np.float32(np.nan), q), dev), *s.cache, s.plan(), SCALE)
    check_but(o, ref, size, lost)


def test_attention_nan_keys_of_whole_items_reach_the_result(pkg, dev):
    """The keys of a sequence's first four items out of eight, which a lane of the merge loads at once, are NaN."""
    s = Step(pkg, dev, [2000] * 16, [1] * 16, 32, 4, seed=41)
    s.k[s.ref[4][3, :64]] = 0x7F
    s.cache = (torch.from_numpy(s.k).to(dev).view(FP8), *s.cache[1:])
    q = orc.round_bf16(s.rng.standard_normal((s.T, 32, D)).astype(np.float32))
    ref, size = s.attention_ref(q)
    lost = np.zeros((s.T, 32, 1), bool)
    lost[3] = True
    check_but(pkg.paged_attention_fp8(to_bf16(q, dev), *s.cache, s.plan(), SCALE), ref, size, lost)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -3.0])
@pytest.mark.parametrize("cached,new", [([40, 700], [1, 1]), ([20, 100], [1, 30]), ([9000, 64], [1, 1])])
def test_attention_takes_no_scale_of_a_page_that_no_sequence_has(pkg, dev, bad, cached, new):
    """A pool whose scales were never filled: those of pages without an owner, page 0 among them, may be anything, and
    an odd number of pages leaves half a pair and a part of a tile's step without one."""
    s = Step(pkg, dev, cached, new, 32, 4, seed=42)
    up = lambda a: np.where(a >= 0, a + 1, a).astype(np.int32)  # noqa: E731
    s.tables, s.free = up(s.tables), up(s.free)
    s.ref = kv.plan(s.cached, s.new, s.tables, s.free, s.T, s.max_new)
    s.g_tables, s.g_free = i32(s.tables, dev), i32(s.free, dev)
    own = np.unique(s.ref[4][s.ref[4] >= 0])
    pools = [np.concatenate([a[:1], a]) for a in (s.k, s.v, s.ks, s.vs)]
    for a in pools[2:]:
        a[~np.isin(np.arange(len(a)), own)] = bad
    s.cache = tuple(torch.from_numpy(a).to(dev) for a in pools)
    s.cache = (s.cache[0].view(FP8), s.cache[1].view(FP8), *s.cache[2:])
    with np.errstate(invalid="ignore"):  # the oracle unpacks these pages, too
        s.check_attention(s.plan())


LATE = [
    ([70], [5], 8, 4, None),             # 10 rows
    ([9000, 30], [4, 2], 8, 2, None),    # 16 rows, split
    ([40, 0], [150, 33], 32, 4, None),   # tiles
    ([3000], [40], 32, 4, None),         # tiles, split
    ([100], [300], 64, 4, 2100),         # tiles of 256 rows
]


@pytest.mark.parametrize("cached,new,Hq,Hkv,T", LATE)
def test_attention_nan_reaches_no_earlier_token(pkg, dev, cached, new, Hq, Hkv, T):
    """A NaN in K or V of a step's own token: in the rows from that token on, of V in its dim alone."""
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=43, T=T)
    q = orc.round_bf16(s.rng.standard_normal((s.T, Hq, D)).astype(np.float32))
    ref, size = s.attention_ref(q)
    k, v, lost, G = s.k.copy(), s.v.copy(), np.zeros((s.T, Hq, D), bool), Hq // Hkv
    for i, n in ((0, new[0] // 2), (len(new) - 1, new[-1] - 1)):
        t = int(s.ref[2][i]) + n
        page, slot = divmod(int(s.ref[1][t]), PAGE)
        v[(page, 0, *kv.v_index(slot, np.array([3, 77])))] = 0x7F, 0xFF
        k[(page, 1, *kv.k_index(slot, np.array([100])))] = 0x7F
        rows = slice(t, int(s.ref[2][i + 1]))
        lost[rows, :G, [[3], [77]]] = True
        lost[rows, G:2 * G] = True
    s.cache = (torch.from_numpy(k).to(dev).view(FP8), torch.from_numpy(v).to(dev).view(FP8), *s.cache[2:])
    check_but(pkg.paged_attention_fp8(to_bf16(q, dev), *s.cache, s.plan(), SCALE), ref, size, lost)


@pytest.mark.parametrize("cached,new,Hq,Hkv,T", LATE)
def test_attention_values_past_the_largest_reach_no_earlier_token(pkg, dev, cached, new, Hq, Hkv, T):
    """A value within half a code of 2^128 is coded as 2^128, which is infinite in 32 bits, and so is an infinity
    beside it: not to be multiplied by the zero probabilities of the rows before it."""
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=44, T=T)
    t = new[0] // 2
    k, v = new_kv(s)
    v[t, 1, 5], v[t, 1, 9] = 3.38e38, -np.inf
    p = s.plan()
    pkg.kv_append_fp8(to_bf16(k, dev), to_bf16(v, dev), *s.cache, p)
    q = orc.round_bf16(s.rng.standard_normal((s.T, Hq, D)).astype(np.float32))
    with np.errstate(all="ignore"):
        gk, gv, ks, vs = s.got()
        clean = kv.unpack(gv, vs, kv.v_index)
        past = np.abs(clean) >= 2.0 ** 128
        assert past.sum() == 2
        ref, size = kv.attention(q, kv.unpack(gk, ks, kv.k_index), np.where(past, 0, clean), s.ref[2], s.ref[0], s.ref[4],
                                 SCALE)
    lost, G = np.zeros((s.T, Hq, D), bool), Hq // Hkv
    lost[t:new[0], G:2 * G, [[5], [9]]] = True
    check_but(pkg.paged_attention_fp8(to_bf16(q, dev), *s.cache, p, SCALE), ref, size, lost)


@pytest.mark.parametrize("T,Hq,Hkv", [(9000, 16, 1), (2100, 64, 4), (11000, 12, 4), (9400, 14, 2)])
def test_attention_large_step_mostly_padding(pkg, dev, T, Hq, Hkv):
    """A step of a large capacity that holds a chunk and a few single tokens: tiles of 256 rows (of 255 and 252, where
    the group does not divide them), few enough to be split along their keys."""
    s = Step(pkg, dev, [3000, 700, 0, 5], [300, 1, 2, 0], Hq, Hkv, seed=45, T=T, max_new=2000)
    s.check_attention(s.plan())


@pytest.mark.parametrize("T,Hq,Hkv", [(600, 32, 4), (2100, 64, 4)])
def test_attention_decode_steps_under_a_chunks_capacity(pkg, dev, T, Hq, Hkv):
    """A graph captured for chunks, replayed on 120 decoding sequences alone, then on a chunk with 40 of them, then on
    nothing: the short items run beside no tiles, beside some, and not at all."""
    rng = np.random.default_rng(46)
    B = 120
    cached = [int(c) for c in rng.integers(1, 1500, B)]
    s = Step(pkg, dev, cached, [1] * B, Hq, Hkv, seed=46, T=T, max_new=400, width=300, spare=40)
    held = {}

    def step():
        held["plan"] = s.plan()
        held["o"] = pkg.paged_attention_fp8(held["q"], *s.cache, held["plan"], SCALE)

    q = orc.round_bf16(rng.standard_normal((T, Hq, D)).astype(np.float32))
    held["q"] = to_bf16(q, dev)
    g_tables = s.g_tables.clone()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    plan, o = held["plan"], held["o"]
    for new in ([1] * B, [400] + [1] * 40 + [0] * (B - 41), [0] * B):
        s.new = new
        s.ref = kv.plan(s.cached, new, s.tables, s.free, T, s.max_new)
        s.g_new.copy_(i32(new, dev))
        s.g_tables.copy_(g_tables)
        o.fill_(7)
        graph.replay()
        s.check_plan(plan)
        s.check_output(o, q)
        again = s.plan()
        assert torch.equal(o, pkg.paged_attention_fp8(held["q"], *s.cache, again, SCALE))


@pytest.mark.parametrize("cached,new", [([131000, 100001], [1, 3]), ([100000], [40]), ([120000, 60], [33, 1])])
def test_attention_far_contexts(pkg, dev, cached, new):
    s = Step(pkg, dev, cached, new, 16, 1, seed=47)
    s.check_attention(s.plan())


@pytest.mark.parametrize("cached,new", [*LENS, ([100000, 131000], [3, 1]), ([0, 60000], [700, 500])])
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (14, 2), (5, 5)])
def test_qk_norm_rope_append_keys_to_the_bit(pkg, dev, cached, new, Hq, Hkv):
    """Codes and scales of K where pages begin and go on, for group sizes and positions other than the above."""
    s = Step(pkg, dev, cached, new, Hq, Hkv, seed=48, T=sum(new) + 2)
    x = orc.round_bf16(s.rng.standard_normal((s.T, Hq + 2 * Hkv, D)).astype(np.float32))
    qw, kw = (orc.round_bf16((1 + 0.3 * s.rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    inv_freq = (1e6 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
    pkg.qk_norm_rope_append_fp8(to_bf16(x.reshape(s.T, -1), dev), to_bf16(qw, dev), to_bf16(kw, dev),
                                torch.from_numpy(inv_freq).to(dev), Hq, Hkv, 1e-6, *s.cache, s.plan())
    k, _ = kv.norm_rope(x[:, Hq:Hq + Hkv], kw, inv_freq, s.ref[0], float(np.float32(1e-6)))
    ek, eks = s.k.copy(), s.ks.copy()
    kv.append(k, s.ref[1], s.ref[0], ek, eks, kv.k_index)
    gk, _, gks, _ = s.got()
    assert np.array_equal(gks, eks)
    assert np.array_equal(gk & 127, ek & 127) and np.array_equal(gk[(ek & 127) != 0], ek[(ek & 127) != 0])


@pytest.mark.parametrize("cached,new", [([300, 420, 900], [1, 1, 2]), ([6000, 2000], [1, 1]), ([300], [40])])
def test_attention_of_one_key_is_its_value(pkg, dev, cached, new):
    """Rows of which one key has almost all the weight, a probability that bf16 does not hold: the sum has to be of the
    probabilities as they are multiplied, so that the rounding cancels.  |sum p d (v - o)| <= 2^-8 sum p |v - o|, the mean
    distance, which is at most the standard deviation of V under p (5% more as in the module's bound), and the output's
    rounding; no 2^-8 of the value itself for p."""
    H = 8
    s = Step(pkg, dev, cached, new, H, H, seed=49)
    sign = np.where(s.rng.integers(0, 2, (H, D)) > 0, 1.0, -1.0)
    steps = np.array([0.28125, 0.3125, 0.34375, 0.375, 0.40625, 0.4375, 0.46875, 0.25])  # 4 to 7.7 in the power of 2
    s.ks[:] = 1
    for b in range(len(cached)):
        c = np.full((s.width * PAGE, H), -2.0)
        c[0], c[256 + 3] = 0, steps  # of one wave, the second after the first has set what the others are measured by
        for j, page in enumerate(s.ref[4][b]):
            for slot in range(PAGE if page >= 0 else 0):
                row = kv.to_e4m3(c[j * PAGE + slot][:, None] * sign).T
                s.k[(page, slice(None), *kv.k_index(slot, np.arange(D)))] = row
    s.cache = (torch.from_numpy(s.k).to(dev).view(FP8), s.cache[1], torch.from_numpy(s.ks).to(dev), s.cache[3])
    q = np.broadcast_to(sign, (s.T, H, D)).astype(np.float32)
    k, v, ks, vs = s.got()
    k, v = kv.unpack(k, ks, kv.k_index), kv.unpack(v, vs, kv.v_index)
    ref, size = kv.attention(q, k, v, s.ref[2], s.ref[0], s.ref[4], SCALE)
    square, _ = kv.attention(q, k, v * v, s.ref[2], s.ref[0], s.ref[4], SCALE)
    apart = np.sqrt(np.maximum(square - ref * ref, 0))
    got = pkg.paged_attention_fp8(to_bf16(q, dev), *s.cache, s.plan(), SCALE).float().cpu().numpy()
    worst = np.abs(got - ref) - 2.0 ** -8 * (1.05 * apart + np.abs(ref)) - 2.0 ** -16 * (size + np.abs(ref))
    assert (worst <= 1e-30).all(), (worst.max(), np.argwhere(worst > 0)[:4])
