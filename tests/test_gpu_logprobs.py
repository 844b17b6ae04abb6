"""Log probabilities, entropy and most likely tokens on the GPU against their definition in 64 bits.

Tolerances, from the roundings alone.  A term of Z is 2^d, with d = (x - m) log2(e) off by 2^-24 of it and by the 2^-25 that
log2(e) is off in fp32, and the exponential by 2^-23; the terms that make up Z have |d| below 32 (what is below 2^-32 of
them weighs as little), so each is off by at most (32 * 0.7 * 1.5 + 2) * 2^-24, below 36 * 2^-24, of its value.  A lane
sums at most V / 256 + 9 of them, and 8 joins follow.  In all Z, and so ln Z, is off by at most
  z = (60 + V / 256) * 2^-24.
A logprob is off by that and its rounding.  The entropy, ln Z - (sum e^(x-m) (x-m)) / Z, by z, and by 2 z of the second part,
whose terms are of one sign but for those up to 5.5 above the reference: with D = sum p |x - m|, z (1 + 2 (D + 11)).  Ids are exact."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def top_ref(x, k):
    """NaN first, then descending, the lower index first among equals."""
    key = np.where(np.isnan(x), np.inf, x)
    nan_first = np.where(np.isnan(x), 0, 1)
    return np.stack([np.lexsort((np.arange(x.shape[1]), -row, first))[:k] for row, first in zip(key, nan_first)])


def check(pkg, logits, tokens, k):
    r = pkg.token_logprobs(logits, tokens, k)
    x = logits.double().cpu()
    T, V = x.shape
    z = (60 + V / 256) * 2.0 ** -24
    want = torch.log_softmax(x, 1)
    p = want.exp()
    dist = (p * (x - x.amax(1, keepdim=True)).abs().nan_to_num(posinf=0.0)).sum(1)
    entropy = -(p * torch.where(p > 0, want, 0.0)).sum(1)
    entropy = torch.where(want.isnan().any(1), NAN, entropy)

    def near(got, ref, tol):
        got, ref = got.double().cpu(), ref
        same = (got == ref) | (got.isnan() & ref.isnan())
        assert (same | ((got - ref).abs() <= tol)).all(), (got - ref).abs().max()

    near(r.entropy, entropy, z * (1 + 2 * (dist + 11)) + 2.0 ** -23 * entropy.abs())
    if tokens is not None:
        g = tokens.cpu().long()
        ref = want[torch.arange(T), g.clamp(0, V - 1)]
        ref = torch.where(g < 0, 0.0, torch.where(g < V, ref, NAN))
        near(r.logprobs, ref, z + 2.0 ** -23 * ref.abs())
    else:
        assert r.logprobs is None
    assert r.top_ids.shape == r.top_logprobs.shape == (T, k)
    if k:
        ids = torch.from_numpy(top_ref(x.numpy(), k))
        assert torch.equal(r.top_ids.cpu(), ids)
        ref = want.gather(1, ids)
        near(r.top_logprobs, ref, z + 2.0 ** -23 * ref.abs())
    return r


def logits_of(dev, T, V, dtype=torch.bfloat16, seed=0, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn((T, V + pad), generator=g, device=dev) * 3).to(dtype)[:, pad:]


def tokens_of(dev, T, V, seed=0, dtype=torch.int64):
    return torch.randint(-1, V, (T,), generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(1, 1), (2, 3), (1, 7), (3, 8), (5, 100), (2, 513), (7, 2048), (1, 4096), (2, 4097),
                                 (64, 1000), (3, 32003), (1, 151936), (70, 50257), (1100, 2500)])
def test_sizes(pkg, dev, T, V, dtype):
    for k in sorted({0, 1, min(V, 5), min(V, 64)}):
        check(pkg, logits_of(dev, T, V, dtype, seed=T + V), tokens_of(dev, T, V), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [1, 3, 5, 8])
@pytest.mark.parametrize("V", [5, 1000, 9001])
def test_rows_apart_at_any_address(pkg, dev, V, pad, dtype):
    check(pkg, logits_of(dev, 6, V, dtype, seed=pad, pad=pad), tokens_of(dev, 6, V), min(V, 9))


def test_tokens_of_either_type_or_none(pkg, dev):
    x = logits_of(dev, 6, 700)
    t = torch.tensor([0, 699, -1, -100, 700, 1 << 30], device=dev)
    a, b = check(pkg, x, t, 2), check(pkg, x, t.int(), 2)
    assert torch.equal(a.logprobs[:4], b.logprobs[:4]) and a.logprobs[2:4].tolist() == [0.0, 0.0] and a.logprobs[4:].isnan().all()
    check(pkg, x, None, 2)
    far = torch.tensor([1 << 40, -(1 << 40), 5, 5, 5, 5], device=dev)  # not their low 32 bits
    got = pkg.token_logprobs(x, far).logprobs
    assert got[0].isnan() and got[1] == 0


# Rows of every kind in one batch, split over workgroups (few rows) and not (many)
def odd_rows(V, dtype):
    lowest = torch.finfo(dtype).min
    rng = np.random.default_rng(V)
    base = rng.normal(size=V) * 3

    def row(*parts):
        x = base.copy()
        for first, end, value in parts:
            x[first:end] = value
        return x

    half, third = V // 2, V // 3
    rows = [
        base, np.zeros(V), np.full(V, -INF), np.full(V, lowest), np.full(V, NAN), np.full(V, INF),
        np.sort(base), np.sort(base)[::-1], np.arange(V) % 3,
        row((0, 1, NAN)), row((V - 1, V, NAN)), row((half, half + 1, INF)), row((half, half + 1, INF), (third, third + 1, NAN)),
        row((0, V - 3, -INF)), row((3, V, -INF)), row((0, half, -INF)), row((0, V - 3, lowest)), row((half, V, lowest)),
        row((0, half, -INF), (half, half + 9, NAN)), row((third, third + 2, -NAN), (half, half + 1, -INF)),
        base * 1e4, base * 1e30, base * 0 - 1e37, base + 2e5, row((third, third + 2, 3e38)),
        np.where(np.arange(V) % 2, 0.0, -0.0), row((third, third + 1, 60.0)),
        np.where(np.arange(V) < 5, 3.0, -INF), np.where(np.arange(V) % 7 == 0, 8.0, base),
    ]
    return torch.from_numpy(np.stack(rows)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [64, 1500, 20001])
@pytest.mark.parametrize("copies", [1, 40])
def test_odd_rows(pkg, dev, V, dtype, copies):
    x = odd_rows(V, dtype).repeat(copies, 1).to(dev)
    n = len(x)
    for k in (0, 3, 64):
        check(pkg, x, tokens_of(dev, n, V, seed=k), k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_long_row_of_ties(pkg, dev, dtype):
    """More candidates than are kept: equal values, and values that rise to the row's end."""
    V = 140000
    x = torch.stack([torch.full((V,), 2.0), torch.linspace(-9, 9, V), (torch.arange(V) // 1000).float(),
                     torch.where(torch.arange(V) > V - 300, 5.0, torch.linspace(-3, 4, V))]).to(dtype).to(dev)
    check(pkg, x, tokens_of(dev, 4, V), 64)
    check(pkg, x.repeat(300, 1), tokens_of(dev, 1200, V), 20)


def test_far_rows_of_a_large_batch(pkg, dev):
    """Offsets past 2^32 bytes and 2^31 values."""
    T, V = 15000, 151936
    x = torch.zeros((T, V), dtype=torch.bfloat16, device=dev)
    x[-3:] = logits_of(dev, 3, V)
    tokens = tokens_of(dev, T, V)
    r = pkg.token_logprobs(x, tokens, 4)
    part = check(pkg, x[-3:].clone(), tokens[-3:], 4)
    for a, b in zip(r, part):  # the same values, whether a row is split or not: to fp32's rounding
        assert torch.allclose(a[-3:].double(), b.double(), rtol=2e-5, atol=2e-5)
    assert torch.allclose(r.entropy[:-3], torch.tensor(math.log(V), device=dev), rtol=2e-5)
    assert torch.equal(r.top_ids[0], torch.arange(4, device=dev))


def test_no_rows(pkg, dev):
    r = pkg.token_logprobs(torch.empty((0, 9), device=dev), torch.empty(0, dtype=torch.int64, device=dev), 3)
    assert r.logprobs.shape == r.entropy.shape == (0,) and r.top_ids.shape == (0, 3)


def test_one_row_of_a_wide_stride(pkg, dev):
    x = logits_of(dev, 1, 500, pad=4)
    check(pkg, x, tokens_of(dev, 1, 500), 5)
    check(pkg, x.repeat(3, 1).as_strided((2, 400), (500, 1)), tokens_of(dev, 2, 400), 5)


@pytest.mark.parametrize("T,k", [(1, 5), (40, 20), (1200, 3)])
def test_graph_replays(pkg, dev, T, k):
    V = 30000
    x, t = logits_of(dev, T, V), tokens_of(dev, T, V)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.token_logprobs(x, t, k)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = pkg.token_logprobs(x, t, k)
    for seed in range(4):
        x.copy_(logits_of(dev, T, V, seed=50 + seed))
        t.copy_(tokens_of(dev, T, V, seed=seed))
        want = pkg.token_logprobs(x, t, k)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_two_streams_at_once(pkg, dev):
    xs = [logits_of(dev, 30, 60000, seed=s) for s in range(2)]
    want = [pkg.token_logprobs(x, None, 10) for x in xs]
    torch.cuda.synchronize()
    got = []
    for x in xs:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(pkg.token_logprobs(x, None, 10))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a[1:], b[1:]))


def test_refusals(pkg, dev):
    x, t = logits_of(dev, 4, 100), torch.zeros(4, dtype=torch.int64, device=dev)
    for args in ((x[0],), (x, t[:3]), (x, t, 101), (x, t, -1), (x.repeat(1, 2), t, 65), (x.T, None), (x[:, :0], None),
                 (x, t[None]), (x.cpu(), None), (x, t.cpu()), (x[:1].expand(4, 100), t)):
        with pytest.raises(ValueError):
            pkg.token_logprobs(*args)
    for args in ((x.half(),), (None,), (x, t.float()), (x, [0])):
        with pytest.raises(TypeError):
            pkg.token_logprobs(*args)


@pytest.mark.parametrize("T,k", [(3, 7), (900, 20)])
def test_rows_that_rise_and_fall(pkg, dev, T, k):
    """Candidates keep coming along a row that rises, in one wave's places alone, or in steps; none after the first values of
    one that falls."""
    V = 60000
    at = torch.arange(V, dtype=torch.float32)
    wave = torch.where(at // 512 % 4 == 1, at / V * 9, -5.0)
    rows = torch.stack([at / V * 9 + at % 7 * 1e-3, wave, (at // 4096) * 0.75 - at % 3, 9 - at / V * 9])
    x = torch.cat([rows.to(torch.bfloat16), rows[:, torch.randperm(V, generator=torch.Generator().manual_seed(1))].to(torch.bfloat16)]).to(dev)
    x = x.repeat((T + 7) // 8, 1)[:T].contiguous()
    r = check(pkg, x[:8].contiguous(), tokens_of(dev, min(T, 8), V), k)
    many = pkg.token_logprobs(x, None, k)
    assert torch.equal(many.top_ids[:8], r.top_ids) and torch.equal(many.top_ids[-1], r.top_ids[(T - 1) % 8])
    check(pkg, x.float()[:8].contiguous(), None, k)


@pytest.mark.parametrize("dtype,stride", [(torch.bfloat16, (1 << 31) + 8), (torch.float32, (1 << 30) + 3)])
def test_rows_2_31_apart(pkg, dev, dtype, stride):
    T, V = 3, 5000
    whole = torch.empty((T - 1) * stride + V, dtype=dtype, device=dev)
    x = whole.as_strided((T, V), (stride, 1))
    x.copy_(logits_of(dev, T, V, dtype))
    check(pkg, x, tokens_of(dev, T, V), 6)


def test_a_row_of_2_27(pkg, dev):
    """One row in 64 parts, its largest at the edges and in the middle.  Tolerances as above, for a lane's 2^13 values."""
    V = (1 << 27) + 5
    x = logits_of(dev, 1, V)
    for at, v in ((V - 1, 24.0), (0, 23.0), (V // 2, 22.0), (V - 6, 21.0)):
        x[0, at] = v
    r = pkg.token_logprobs(x, torch.tensor([V - 1], device=dev), 4)
    d = x[0].double()
    ln_z = d.logsumexp(0)
    entropy = ln_z - ((d - ln_z).exp() * d).sum()
    z = (60 + V / 64 / 256) * 2.0 ** -24
    assert r.top_ids.tolist() == [[V - 1, 0, V // 2, V - 6]]
    assert (r.top_logprobs[0].double() - torch.tensor([24.0, 23, 22, 21], device=dev) + ln_z).abs().max() <= z + 2.0 ** -22
    assert r.logprobs[0] == r.top_logprobs[0, 0]
    dist = (24 * torch.ones((), device=dev) - (ln_z - entropy)).abs().double()
    assert (r.entropy[0].double() - entropy).abs() <= z * (1 + 2 * (dist + 11)) + 2.0 ** -23 * entropy.abs()


@pytest.mark.parametrize("mask", [-INF, -1e9, -3.3895313892515355e38])
@pytest.mark.parametrize("T,V,k", [(1, 151936, 20), (40, 20001, 5), (900, 9000, 64)])
def test_masked_rows(pkg, dev, T, V, k, mask):
    """A mask that leaves 3, k - 1, k or many tokens, at the row's start, its end or anywhere; among equals the first ones."""
    g = torch.Generator().manual_seed(T)
    x = torch.full((8, V), mask)
    for i, n in enumerate((3, k - 1, k, 1000)):
        places = torch.randperm(V, generator=g)[:n]
        x[i, places] = torch.randn(n, generator=g) * 3
        at = n if i % 2 else V - n
        x[4 + i, at - n if i % 2 else at:at if i % 2 else V] = torch.randn(n, generator=g) * 3
    x = x.to(torch.bfloat16).to(dev)
    tokens = torch.stack([row.argmax() for row in x])
    few = check(pkg, x[:min(T, 8)].contiguous(), tokens[:min(T, 8)], k)
    check(pkg, x[:2].float().contiguous(), None, k)
    if T > 8:
        many = pkg.token_logprobs(x.repeat((T + 7) // 8, 1)[:T].contiguous(), None, k)
        for i in range(8):
            assert torch.equal(many.top_ids[i::8], few.top_ids[i:i + 1].expand(many.top_ids[i::8].shape))


def test_rows_far_below_zero(pkg, dev):
    """Maxima on both sides of where a reference times log2(e) is no longer held closely, and parts of a row far below the rest."""
    V = 9001
    g = torch.Generator().manual_seed(3)
    near = torch.randn(V, generator=g)
    at = torch.arange(V)
    rows = [near - 726817 + off for off in (-400, -200, -3, 0, 3, 200, 400)]
    rows += [torch.where(at // 512 % 4 == 1, near, near - 1e6), torch.where(at < V // 2, near - 5e8, near),
             torch.where(at % 2 == 0, near - 726600, near - 726900), torch.where(at == V - 1, 0.0, near - 3e38)]
    x = torch.stack(rows).to(dev)
    check(pkg, x, tokens_of(dev, len(rows), V), 9)
    check(pkg, x.repeat(80, 1), tokens_of(dev, 80 * len(rows), V), 9)


@pytest.mark.parametrize("T,V,k", [(1, 151936, 20), (3, 3000, 64), (40, 20001, 5), (900, 9000, 64)])
def test_rows_of_few_values(pkg, dev, T, V, k):
    """Among thousands of equals the first ones: all the same, of two or five values, the larger ones at the end alone, a step
    down, runs along the row."""
    g = torch.Generator().manual_seed(V)
    at = torch.arange(V)
    x = torch.stack([torch.zeros(V), torch.randint(0, 2, (V,), generator=g).float(), torch.randint(-2, 3, (V,), generator=g).float(),
                     (at > V - k // 2 - 2).float(), (at < V // 3).float(), (at // 777 % 3).float(),
                     torch.where(at // 512 % 4 == 2, 1.0, 0.0), torch.where(torch.rand(V, generator=g) < 2 * k / V, 1.0, 0.0)])
    x = x.to(torch.bfloat16).to(dev)
    n = min(T, 8)
    few = check(pkg, x[:n].contiguous(), tokens_of(dev, n, V), k)
    check(pkg, x[-n:].float().contiguous(), None, k)
    check(pkg, x[-n:].contiguous(), None, 1)
    if T > 8:
        many = pkg.token_logprobs(x.repeat((T + 7) // 8, 1)[:T].contiguous(), None, k)
        for i in range(8):
            assert torch.equal(many.top_ids[i::8], few.top_ids[i:i + 1].expand(many.top_ids[i::8].shape))
