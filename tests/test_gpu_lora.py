"""Adapters beside a shared projection on the GPU: the plan of a step's rows against a stable sort, what the adapters add
against the formula in 64 bits.

Tolerance of an output, from the roundings alone: the result's own, half a bf16 step, 2^-8 of it; A x summed in fp32, off
by K * 2^-24 of the sum of its terms' sizes, and kept as two bf16 values, off by 2^-17 of it; the second sum of 2 R terms
and y in fp32.  With S = scale * sum_r (sum_k |x a|) |b|, all but the first are at most
(K + 2 R + 2) * 2^-24 * (S + |y|) + 2^-17 * S."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plan_ref(ids, L, cu=None, T=None):
    if cu is not None:
        rows = np.full(T, -1)
        for b, i in enumerate(ids):
            rows[min(cu[b], T):min(cu[b + 1], T)] = i
        ids = rows
    key = np.where((np.asarray(ids) >= 0) & (np.asarray(ids) < L), ids, L)
    return np.argsort(key, kind="stable"), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=L + 1))])


def i32(a, dev):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def lists_of(plan):
    """The plan's tiles of 64 rows and of 2, as the kernels read them, and the room for each."""
    buf = plan.buffer.cpu().numpy()
    T, some = plan.num_rows, min(plan.num_rows, plan.num_adapters)
    at = (plan._at[1] + T + 3) // 4 * 4
    rooms = (T // 64 + some, T // 2 + some if T <= 256 else 0)
    assert len(buf) == at + 4 * sum(rooms)
    return [(buf[a:a + 4 * n].reshape(-1, 4), n, room) for a, n, room in ((at, buf[0], rooms[0]), (at + 4 * rooms[0], buf[1] if rooms[1] else 0, rooms[1]))]


@pytest.mark.parametrize("T,L", [(0, 1), (1, 1), (1, 256), (5, 3), (63, 2), (64, 256), (65, 100), (1000, 7), (1024, 1),
                                 (1025, 256), (4096, 3), (10000, 40), (70001, 256)])
def test_plan_by_row(pkg, dev, T, L):
    rng = np.random.default_rng(T + L)
    ids = rng.integers(-1, L + 1, T)  # some outside on either side
    if T >= 1000:
        ids[T // 3:T // 2] = L // 2   # a long run, as prompts have
    plan = pkg.lora_plan(i32(ids, dev), L)
    rows, offsets = plan_ref(ids, L)
    assert np.array_equal(plan.rows.cpu().numpy(), rows) and np.array_equal(plan.offsets.cpu().numpy(), offsets)
    for height, (tiles, n, room) in zip((64, 2), lists_of(plan)):
        want = [(l, o, min(height, offsets[l + 1] - o), 0) for l in range(L) for o in range(offsets[l], offsets[l + 1], height)]
        assert n <= room and (not room or np.array_equal(tiles, np.asarray(want).reshape(-1, 4)))


@pytest.mark.parametrize("lens,T", [([3], 3), ([0, 5, 0, 0, 7, 1], 13), ([1] * 64, 64), ([700, 1, 1300, 64], 3000),
                                    ([30, 50], 40), ([2500, 3000], 2600), ([], 9), ([0, 0], 4), ([1] * 4096, 4100)])
def test_plan_by_sequence(pkg, dev, lens, T):
    """Padding behind the last sequence, and sequences past the step's rows, have no adapter."""
    rng = np.random.default_rng(len(lens))
    L = 9
    ids = rng.integers(-1, L + 1, len(lens))
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(int)
    plan = pkg.lora_plan(i32(ids, dev), L, cu_rows=i32(cu, dev), num_rows=T)
    rows, offsets = plan_ref(ids, L, cu, T)
    assert np.array_equal(plan.rows.cpu().numpy(), rows) and np.array_equal(plan.offsets.cpu().numpy(), offsets)


def test_plan_with_rows_in_front_of_the_first_sequence(pkg, dev):
    plan = pkg.lora_plan(i32([1], dev), 2, cu_rows=i32([5, 8], dev), num_rows=10)
    assert plan.rows.tolist() == [5, 6, 7, 0, 1, 2, 3, 4, 8, 9] and plan.offsets.tolist() == [0, 0, 3, 10]


class Case:
    def __init__(self, pkg, dev, T, K, columns, R, ranks, seed=0, x_pad=0, y_pad=0, ids=None, poison=False):
        g = torch.Generator(device=dev).manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
        L, N, P = len(ranks), sum(columns), len(columns)
        self.T, self.K, self.R, self.columns, self.ranks = T, K, R, columns, ranks
        self.x = n(T, K + x_pad).to(torch.bfloat16)[:, x_pad:]
        self.y = n(T, N + y_pad).to(torch.bfloat16)[:, :N]
        self.a = (n(L, P * R, K) * K ** -0.5).to(torch.bfloat16)
        self.b = (n(L, N, R) * 0.1).to(torch.bfloat16)
        self.scales = torch.rand((L,), generator=g, device=dev) * 3
        if poison:  # what lies past an adapter's rank may be anything
            for l, r in enumerate(ranks):
                self.a[l].view(P, R, K)[:, max(r, 0):] = float("nan")
                self.b[l, :, max(r, 0):] = float("nan")
        self.ids = np.random.default_rng(seed).integers(-1, L, T) if ids is None else np.asarray(ids)
        self.pool = pkg.LoraPool(self.a, self.b, i32(ranks, dev), self.scales, columns)
        self.plan = pkg.lora_plan(i32(self.ids, dev), L)

    def expected(self):
        """(values, sizes of the terms) in 64 bits"""
        x, y, a, b = (t.double().cpu() for t in (self.x, self.y, self.a, self.b))
        out, size = y.clone(), torch.zeros_like(y)
        for l, r in enumerate(self.ranks):
            rows, r = np.nonzero(self.ids == l)[0], min(r, self.R)
            if r <= 0 or not len(rows):
                continue
            s, n0 = float(self.scales[l]), 0
            for p, n in enumerate(self.columns):
                al, bl = a[l, p * self.R:p * self.R + r], b[l, n0:n0 + n, :r]
                out[rows, n0:n0 + n] += s * (x[rows] @ al.T) @ bl.T
                size[rows, n0:n0 + n] = s * (x[rows].abs() @ al.abs().T) @ bl.abs().T
                n0 += n
        return out, size

    def check(self, got):
        want, size = self.expected()
        tol = 2.0 ** -8 * want.abs() + (self.K + 2 * self.R + 2) * 2.0 ** -24 * (size + self.y0.double().cpu().abs()) + 2.0 ** -17 * size
        assert ((got.double().cpu() - want).abs() <= tol).all()
        alone = ~np.isin(self.ids, [l for l, r in enumerate(self.ranks) if r > 0])
        assert torch.equal(got[alone], self.y0[alone])

    def run(self, pkg):
        self.y0 = self.y.clone()
        want, size = self.expected()
        out = pkg.lora_add(self.y, self.x, self.pool, self.plan)
        assert out is self.y
        self.expected = lambda: (want, size)
        self.check(out)
        return out


QKV = (512, 128, 128)


@pytest.mark.parametrize("T,K,columns,R,ranks", [
    (1, 32, (32,), 16, [16]),
    (1, 2048, (4096, 512, 512), 16, [8, 16]),
    (3, 4096, (2048,), 64, [64, 1, 33]),
    (17, 256, QKV, 32, [32, 0, 7, -3, 40]),
    (64, 96, (96, 32), 48, [48, 17, 16, 5] * 30),
    (100, 160, (64, 32, 32, 2080), 128, [128, 100, 64, 3]),
    (257, 512, QKV, 80, [80, 65]),
    (1000, 512, QKV, 64, [64]),
    (1100, 256, QKV, 16, [16, 9, 12]),
    (2500, 320, (1056,), 32, [32, 16, 4] * 20),
    (3000, 256, QKV, 128, [128, 64]),
    (5000, 64, (64,), 64, [31, 64]),
])
def test_add(pkg, dev, T, K, columns, R, ranks):
    Case(pkg, dev, T, K, columns, R, ranks, seed=T + K).run(pkg)


@pytest.mark.parametrize("T", [40, 1500])
@pytest.mark.parametrize("R", [16, 64])
def test_past_the_rank_and_rows_apart(pkg, dev, T, R):
    Case(pkg, dev, T, 128, QKV, R, [R, 3, R - 1, 0], seed=R, x_pad=24, y_pad=8, poison=True).run(pkg)


@pytest.mark.parametrize("T", [1, 33, 1100])
def test_one_adapter_and_none(pkg, dev, T):
    Case(pkg, dev, T, 128, QKV, 16, [16, 16], ids=[1] * T).run(pkg)
    c = Case(pkg, dev, T, 128, QKV, 16, [16, 16], ids=[-1, 2] * (T // 2) + [7] * (T % 2))
    before = c.y.clone()
    assert torch.equal(pkg.lora_add(c.y, c.x, c.pool, c.plan), before)


def test_no_rows(pkg, dev):
    c = Case(pkg, dev, 0, 64, (64,), 16, [16])
    assert pkg.lora_add(c.y, c.x, c.pool, c.plan).shape == (0, 64)


@pytest.mark.parametrize("T", [50, 1200])
def test_what_is_not_finite_keeps_to_its_row(pkg, dev, T):
    clean = Case(pkg, dev, T, 128, QKV, 16, [16, 16], seed=3, ids=[0, 1] * (T // 2))
    other = Case(pkg, dev, T, 128, QKV, 16, [16, 16], seed=3, ids=[0, 1] * (T // 2))
    other.x[7, 5] = float("nan")
    other.x[8, 100] = float("inf")
    a, b = pkg.lora_add(clean.y, clean.x, clean.pool, clean.plan), pkg.lora_add(other.y, other.x, other.pool, other.plan)
    rest = [t for t in range(T) if t not in (7, 8)]
    assert torch.equal(a[rest], b[rest]) and b[7].isnan().all() and not b[8].isfinite().any()


def test_an_intermediate_past_bf16(pkg, dev):
    """A x of 3.4e38 rounds to infinity in bf16: the result is that infinity, not NaN."""
    c = Case(pkg, dev, 2, 32, (32,), 16, [1], ids=[0, 0])
    c.x.fill_(2.0 ** 64)
    c.a.fill_(2.0 ** 59)  # 32 terms of 2^123, times the scale
    c.scales.fill_(0.999999)
    c.b.fill_(1.0)
    assert (pkg.lora_add(c.y, c.x, c.pool, c.plan) == float("inf")).all()


def test_pools_are_loaded_and_replaced(pkg, dev):
    g = torch.Generator(device=dev).manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    pool = pkg.LoraPool.empty(3, 64, (96, 32), 32, dev)
    x, y = n(6, 64), n(6, 128)
    plan = pkg.lora_plan(i32([0, 1, 2, 1, 0, -1], dev), 3)
    assert torch.equal(pkg.lora_add(y.clone(), x, pool, plan), y)
    pool.load(1, [(n(32, 64), n(96, 32)), (n(32, 64), n(32, 32))], 1.0)
    parts = [(n(5, 64), n(96, 5)), None]
    pool.load(1, parts, 0.5)  # a smaller one in its place, and one part left alone
    pool.load(2, [None, None], 4.0)
    assert pool.ranks.tolist() == [0, 5, 0]
    out = pkg.lora_add(y.clone(), x, pool, plan)
    assert torch.equal(out[[0, 2, 4, 5]], y[[0, 2, 4, 5]]) and torch.equal(out[:, 96:], y[:, 96:])
    a, b = (t.double() for t in parts[0])
    want = y[1].double()[:96] + 0.5 * (x[1].double() @ a.T) @ b.T
    size = 0.5 * (x[1].double().abs() @ a.abs().T) @ b.abs().T
    assert ((out[1, :96].double() - want).abs() <= 2.0 ** -8 * want.abs() + 130 * 2.0 ** -24 * (size + y[1, :96].double().abs()) + 2.0 ** -17 * size).all()
    for bad in ([parts[0]], [(n(33, 64), n(96, 33)), None], [(n(5, 60), n(96, 5)), None], [(n(5, 64), n(95, 5)), None],
                [(n(5, 64), n(96, 5)), (n(6, 64), n(32, 6))]):
        with pytest.raises(ValueError):
            pool.load(0, bad, 1.0)
    with pytest.raises(ValueError):
        pool.load(3, parts, 1.0)


@pytest.mark.parametrize("T", [48, 1300])
def test_graph_replays_follow_the_adapters(pkg, dev, T):
    """Plan and addition in one graph: replays on other numbers, rows and adapters, each against the eager result."""
    c = Case(pkg, dev, T, 256, QKV, 32, [32, 8, 20], seed=5)
    ids, x, y = i32(c.ids, dev), c.x.clone(), c.y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.lora_add(y, x, c.pool, pkg.lora_plan(ids, 3))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan = pkg.lora_plan(ids, 3)
        pkg.lora_add(y, x, c.pool, plan)
    g = torch.Generator(device=dev).manual_seed(9)
    for _ in range(4):
        ids.copy_(torch.randint(-1, 3, (T,), generator=g, device=dev))
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        y.copy_(torch.randn(y.shape, generator=g, device=dev))
        c.pool.scales.copy_(torch.rand((3,), generator=g, device=dev))
        want = pkg.lora_add(y.clone(), x, c.pool, pkg.lora_plan(ids, 3))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_a_plan_is_filled_again(pkg, dev):
    plan = pkg.lora_plan(i32([0, 1, 0], dev), 2)
    again = pkg.lora_plan(i32([1, -1, 0], dev), 2, out=plan)
    assert again is plan and plan.rows.tolist() == [2, 0, 1] and plan.offsets.tolist() == [0, 1, 2, 3]
    for ids, L in (([0, 1], 2), ([0, 1, 0], 3)):
        with pytest.raises(ValueError):
            pkg.lora_plan(i32(ids, dev), L, out=plan)


def test_two_streams_at_once(pkg, dev):
    cases = [Case(pkg, dev, 700, 512, QKV, 64, [64, 30], seed=s) for s in range(2)]
    want = [pkg.lora_add(c.y.clone(), c.x, c.pool, c.plan) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append(pkg.lora_add(c.y.clone(), c.x, c.pool, pkg.lora_plan(i32(c.ids, dev), 2)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(pkg, dev):
    c = Case(pkg, dev, 8, 64, (64, 32), 16, [16, 4])
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    add = lambda y=c.y, x=c.x, pool=c.pool, plan=c.plan: pkg.lora_add(y, x, pool, plan)  # noqa: E731
    for bad in ({"y": bf(8, 95)}, {"y": bf(7, 96)}, {"x": bf(8, 32)}, {"x": bf(64, 8).T}, {"y": bf(8, 100)[:, :96]},
                {"y": bf(1, 96).expand(8, 96)}, {"plan": pkg.lora_plan(i32([0] * 8, dev), 3)},
                {"plan": pkg.lora_plan(i32([0] * 7, dev), 2)}, {"x": c.x.cpu()}):
        with pytest.raises(ValueError):
            add(**bad)
    for bad in ({"y": c.y.float()}, {"x": None}, {"pool": None}, {"plan": None}):
        with pytest.raises(TypeError):
            add(**bad)
    with pytest.raises(Exception, match="aligned"):
        pkg.lora_add(bf(8 * 96 + 1)[1:].view(8, 96), c.x, c.pool, c.plan)
    ranks, scales = i32([16, 4], dev), torch.ones(2, device=dev)
    pool = lambda a=bf(2, 32, 64), b=bf(2, 96, 16), r=ranks, s=scales, columns=(64, 32): pkg.LoraPool(a, b, r, s, columns)  # noqa: E731
    pool()
    for bad in ({"a": bf(2, 32, 60)}, {"a": bf(2, 16, 64)}, {"b": bf(2, 95, 16)}, {"b": bf(3, 96, 16)}, {"columns": (96,)},
                {"columns": (64, 16, 16)}, {"columns": ()}, {"r": i32([1], dev)}, {"s": torch.ones(3, device=dev)},
                {"a": bf(2, 2 * 144, 64), "b": bf(2, 96, 144)}, {"a": bf(2, 2 * 8, 64), "b": bf(2, 96, 8)}):
        with pytest.raises(ValueError):
            pool(**bad)
    for bad in ({"a": bf(2, 32, 64).float()}, {"r": ranks.long()}, {"s": scales.double()}):
        with pytest.raises(TypeError):
            pool(**bad)
    ids = i32([0] * 4, dev)
    for args in ((ids, 0), (ids, 257), (ids[None], 2), (ids, 2, i32([0, 4], dev), 4), (ids, 2, i32([0, 1, 2, 3, 4], dev)),
                 (ids, 2, i32([0, 1, 2, 3, 4], dev), (1 << 18) + 1), (ids, 2, None, 5)):
        with pytest.raises(ValueError):
            pkg.lora_plan(*args)
    for args in ((ids.long(), 2), ([0], 2)):
        with pytest.raises(TypeError):
            pkg.lora_plan(*args)


@pytest.mark.parametrize("T,K,columns,R,ranks", [
    (16, 8192, (256,), 64, [64]),           # tiles of up to 16 rows, and of more
    (17, 8192, (256,), 64, [64]),
    (65, 8224, (160,), 64, [33]),           # a row over a tile; k past whole slices
    (130, 4128, (288, 32), 80, [80, 1]),
    (256, 2080, (224,), 16, [16] * 256),    # the last step with small tiles, an adapter a row
    (257, 2080, (224,), 16, [16] * 256),
    (128, 2048, (576,), 32, [32, 15]),      # at the limit of the form of few rows, and past it
    (129, 2048, (576,), 32, [32, 15]),
    (90, 8192, (672,), 16, [9] * 40),
    (600, 1312, (96, 96, 96, 96), 112, [112, 97, 65, 64, 63]),
])
def test_edges_of_forms_and_tiles(pkg, dev, T, K, columns, R, ranks):
    Case(pkg, dev, T, K, columns, R, ranks, seed=T + R, ids=[t * len(ranks) // T for t in range(T)]).run(pkg)
    Case(pkg, dev, T, K, columns, R, ranks, seed=T + R, poison=True).run(pkg)


@pytest.mark.parametrize("T,stride", [(40, 512), (1000, 512), (2100, 1 << 21)])
def test_x_and_y_side_by_side(pkg, dev, T, stride):
    """In rows of one buffer, in either order; the longest past 2^32 values."""
    c = Case(pkg, dev, T, 256, (64, 32), 32, [32, 7, 20], seed=2)
    want = pkg.lora_add(c.y.clone(), c.x, c.pool, c.plan)
    whole = torch.empty((T, stride), dtype=torch.bfloat16, device=dev)
    for x, y in ((whole[:, :256], whole[:, 256:352]), (whole[:, -256:], whole[:, -352:-256]), (whole[:, :256], whole[:, -96:])):
        x.copy_(c.x)
        y.copy_(c.y)
        assert torch.equal(pkg.lora_add(y, x, c.pool, c.plan), want) and torch.equal(x, c.x)


@pytest.mark.parametrize("K,N", [(64, 131104), (131104, 64)])
@pytest.mark.parametrize("T", [2, 300])
def test_the_last_adapter_of_a_pool_past_2_32(pkg, dev, K, N, T):
    L, R = 256, 128
    one = Case(pkg, dev, T, K, (N,), R, [128], seed=4, ids=[0] * T)
    a, b = (torch.empty((L, *t.shape[1:]), dtype=t.dtype, device=dev) for t in (one.a, one.b))
    a[-1], b[-1] = one.a[0], one.b[0]
    scales = torch.zeros(L, device=dev)
    scales[-1] = one.scales[0]
    pool = pkg.LoraPool(a, b, i32([0] * (L - 1) + [128], dev), scales, (N,))
    got = pkg.lora_add(one.y.clone(), one.x, pool, pkg.lora_plan(i32([L - 1] * T, dev), L))
    one.run(pkg)
    one.check(got)


def test_an_x_that_it_would_change_is_refused(pkg, dev):
    c = Case(pkg, dev, 8, 64, (64,), 16, [16])
    wide = torch.zeros((9, 192), dtype=torch.bfloat16, device=dev)
    same = torch.zeros((8, 64), dtype=torch.bfloat16, device=dev)
    for y, x in ((same, same), (wide[:8, :64], wide[:8, 56:120]), (wide[:8, :64], wide[1:, :64]), (wide[:8, 128:], wide[:8].flatten()[:512].view(8, 64))):
        with pytest.raises(Exception, match="invalid"):
            pkg.lora_add(y, x, c.pool, c.plan)


@pytest.mark.parametrize("T,R", [(40, 16), (40, 64), (300, 16), (300, 64), (300, 128)])
def test_a_finite_intermediate_past_bf16(pkg, dev, T, R):
    """scale * A x = +-1.999 * 2^127: finite in fp32, past bf16's largest.  Against b of 0, 2^-20, and 1 the result is the formula's,
    whose bf16 is no near tie (1.999 lies 2^-8.4 from the next one)."""
    ids = [0] * (T - 7) + [1] * 7  # tiles of many rows and of few
    c = Case(pkg, dev, T, 32, (96,), R, [R, 1], ids=ids)
    c.x.zero_()
    c.a.zero_()
    c.b.zero_()
    c.x[:, 0] = torch.where(torch.arange(T, device=dev) % 2 == 0, 2.0 ** 64, -(2.0 ** 64))
    c.a[:, 0, 0] = 2.0 ** 63
    c.scales.fill_(1.999)
    c.b[:, 1::3, 0] = 2.0 ** -20
    c.b[:, 2::3, 0] = 1.0
    want = c.expected()[0].float().to(torch.bfloat16)
    got = pkg.lora_add(c.y, c.x, c.pool, c.plan).cpu()
    assert want[:, 2::3].isinf().all() and want[:, 1::3].isfinite().all() and torch.equal(got, want)


@pytest.mark.parametrize("T", [40, 300, 1500])
@pytest.mark.parametrize("R,ranks", [(16, [16, 3]), (32, [20, 32]), (64, [64, 17]), (128, [128, 70])])
def test_infinities_in_b(pkg, dev, T, R, ranks):
    """An infinite value of B makes infinities of its column alone, of the sign of A x, whatever the size of the step; two of
    different signs, and one against a zero, NaN."""
    c = Case(pkg, dev, T, 128, QKV, R, ranks, seed=R, ids=[0] * (T - 9) + [1] * 8 + [-1])
    INF = float("inf")
    c.b[0, 5, 1], c.b[0, 300, 12], c.b[0, 517, 0] = INF, -INF, INF
    c.b[0, 77, 0], c.b[0, 77, 2] = INF, INF
    c.b[1, 6, 2], c.b[1, 767, 0] = -INF, INF
    c.x[4] = 0
    c.y[3, 9], c.y[T - 2, 5], c.y[3, 11] = INF, float("nan"), -INF
    before = c.y.clone()
    want, size = c.expected()
    got = pkg.lora_add(c.y, c.x, c.pool, c.plan).double().cpu()
    odd = ~want.isfinite()
    # per row of the first adapter 4 columns, of the second 2; 3 values of y
    assert odd.sum() == (T - 9) * 4 + 8 * 2 + 3
    assert torch.equal(got[odd].nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))
    tol = 2.0 ** -8 * want.abs() + (c.K + 2 * R + 2) * 2.0 ** -24 * (size + before.double().cpu().abs()) + 2.0 ** -17 * size
    assert ((got - want).abs() <= tol)[~odd].all()
    assert torch.equal(got[-1], before[-1].double().cpu())


@pytest.mark.parametrize("R", [16, 64, 128])
def test_infinities_in_some_pieces_of_a_run(pkg, dev, R):
    """Runs of 512 columns of a long step, some of whose pieces of 128 hold an infinity; tiles of many rows and of few."""
    T = 4200
    c = Case(pkg, dev, T, 128, (4096, 544), R, [R, 7], seed=R, ids=[0] * (T - 9) + [1] * 9, poison=True)
    INF = float("inf")
    for n, r, v in ((200, 0, INF), (511, 3, -INF), (4095, 6, INF), (4096 + 130, 2, INF), (4096 + 543, 1, -INF)):
        c.b[:, n, r] = v
    before = c.y.double().cpu()
    want, size = c.expected()
    got = pkg.lora_add(c.y, c.x, c.pool, c.plan).double().cpu()
    odd = ~want.isfinite()
    assert odd.sum() == T * 5 and torch.equal(got[odd].nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))
    tol = 2.0 ** -8 * want.abs() + (c.K + 2 * R + 2) * 2.0 ** -24 * (size + before.abs()) + 2.0 ** -17 * size
    assert ((got - want).abs() <= tol)[~odd].all()


def form_of(pkg, T, L, K, columns, R):
    """Few rows or many: the form of few rows needs no workspace."""
    import ctypes

    n = pkg._lib.load().moe_mi355x_lora_add_workspace_bytes(T, L, K, R, len(columns), (ctypes.c_int * len(columns))(*columns))
    return "many" if n else "few"


@pytest.mark.parametrize("R", [16, 32, 64, 128])
@pytest.mark.parametrize("paired", [False, True])
def test_few_rows_over_long_runs_of_columns(pkg, dev, R, paired):
    """Runs of 2048 columns, in which a wave has four turns of 64, and a part's last run of fewer; tiles of one row and of two."""
    T, K, columns = 128, 128, (8192, 544, 32)
    ranks = [R, 1, R - 1, 9] * 25
    ids = [t // 2 if paired else t for t in range(T)]
    ids = [i if i < 100 else 99 - i % 100 for i in ids]
    assert form_of(pkg, T, len(ranks), K, columns, R) == "few"
    Case(pkg, dev, T, K, columns, R, ranks, seed=R, ids=ids).run(pkg)
    Case(pkg, dev, T, K, columns, R, ranks, seed=R + 1, ids=ids, x_pad=8, y_pad=24, poison=True).run(pkg)


@pytest.mark.parametrize("R,ranks", [(16, [16, 5]), (32, [32, 17]), (64, [64, 33]), (64, [30, 16]), (128, [128, 65]), (128, [64, 20])])
def test_many_rows_over_long_runs_of_columns(pkg, dev, R, ranks):
    """Runs of 512 columns in four pieces of 128, and a part's last run of fewer; tiles of many rows and of up to 16."""
    T, K, columns = 4100, 256, (4096, 544, 32)
    L = 40
    ranks = (ranks * L)[:L]
    ids = [0] * 2000 + [1] * 1613 + [2 + t // 13 for t in range(494 - 13)]  # the narrow ones of 13 rows
    ids = np.asarray((ids + [-1] * T)[:T])
    assert form_of(pkg, T, L, K, columns, R) == "many"
    Case(pkg, dev, T, K, columns, R, ranks, seed=R, ids=ids).run(pkg)
    Case(pkg, dev, T, K, columns, R, ranks, seed=R + 1, ids=np.random.default_rng(R).permutation(ids), x_pad=8, y_pad=24, poison=True).run(pkg)
