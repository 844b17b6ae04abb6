"""CPU oracle for the 8-bit paged KV cache: a step's plan, the quantising append, q/k norm with rotary, attention.

TEST INFRASTRUCTURE ONLY.  Written from the operators' definitions (``include/moe_mi355x.h``) in plain loops and 64
bits; pinned in ``tests/test_oracle_kv8.py``.  The reference has no counterpart: its cache is contiguous and
unquantised.
"""

from __future__ import annotations

import math

import numpy as np

PAGE, D = 16, 128
MIN_SCALE = 2.0 ** -100


def plan(cached, new, tables, free, T, max_new):
    """(positions [T], slots [T], cu [B + 1], context [B], tables, pages used); tables is a new array."""
    tables = np.array(tables, np.int32)
    B, width = tables.shape
    pos, slot = np.full(T, -1, np.int32), np.full(T, -1, np.int32)
    cu, context, used = [0], [], 0
    for b in range(B):
        c = min(max(int(cached[b]), 0), PAGE * width)
        n = min(min(max(int(new[b]), 0), max_new), T - cu[-1])
        have, total = -(-c // PAGE), min(width, -(-(c + n) // PAGE))
        for j in range(have, total):
            tables[b, j] = free[used] if used < len(free) else -1
            used += 1
        for i in range(n):
            p = c + i
            pos[cu[-1] + i] = p
            if p // PAGE < width and tables[b, p // PAGE] >= 0:
                slot[cu[-1] + i] = tables[b, p // PAGE] * PAGE + p % PAGE
        cu.append(cu[-1] + n)
        context.append(min(c + n, PAGE * width))
    return pos, slot, np.array(cu, np.int32), np.array(context, np.int32), tables, used


def scale_of(amax: float) -> float:
    s = MIN_SCALE
    while amax / s > 448.0:
        s *= 2.0
    return s


def e4m3_values() -> np.ndarray:
    """The 127 non-negative finite e4m3fn values, by code."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return np.array(out)


_VALUES = e4m3_values()
_MIDDLES = (_VALUES[1:] + _VALUES[:-1]) / 2


def to_e4m3(x) -> np.ndarray:
    """Codes of the nearest e4m3 values, ties to even, saturated; NaN is 0x7f with its sign dropped."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    below, above = np.searchsorted(_MIDDLES, a, side="left"), np.searchsorted(_MIDDLES, a, side="right")
    code = np.where(below % 2 == 0, below, above)  # they differ on a tie only: the even one of the two
    code = np.where((below == above) | (below % 2 == 0), code, above)
    return np.where(np.isnan(x), 0x7F, code + 128 * np.signbit(x)).astype(np.uint8)


def from_e4m3(codes) -> np.ndarray:
    codes = np.asarray(codes, np.uint8)
    v = np.append(_VALUES, np.nan)[codes & 127]
    return np.where(codes & 128, -v, v)


def k_index(t, d):
    return d // 16, t, d % 16


def v_index(t, d):
    return d // 64, t // 4, d % 64, t % 4


def append(x, slots, positions, codes, scale, index):
    """Quantises x [T, Hkv, 128] into a pool's ``codes`` (uint8) and ``scale``, in place; ``index``: k_index or v_index."""
    x = np.asarray(x, np.float64)
    d = np.arange(D)
    by_page: dict[int, list[int]] = {}
    for t, s in enumerate(slots):
        if 0 <= s < PAGE * len(codes):
            by_page.setdefault(int(s) // PAGE, []).append(t)
    for page, tokens in by_page.items():
        fresh = any(slots[t] % PAGE == 0 for t in tokens)
        for g in range(x.shape[1]):
            a = np.abs(x[tokens, g])
            need = scale_of(float(np.max(np.where(np.isfinite(a), a, 0.0))))
            s = need if fresh else max(float(scale[page, g]), need)
            old = from_e4m3(codes[page, g])
            codes[page, g] = 0 if fresh else to_e4m3(old * (float(scale[page, g]) / s))
            for t in tokens:
                with np.errstate(invalid="ignore"):
                    codes[(page, g, *index(slots[t] % PAGE, d))] = to_e4m3(x[t, g] / s)
            scale[page, g] = s


def unpack(codes, scale, index) -> np.ndarray:
    """[pages, Hkv, 16, 128] values."""
    out = np.empty((*codes.shape[:2], PAGE, D))
    v = from_e4m3(codes)
    for t in range(PAGE):
        out[:, :, t, :] = v[(slice(None), slice(None), *index(t, np.arange(D)))]
    return out * np.asarray(scale, np.float64)[..., None, None]


def norm_rope(x, weight, inv_freq, positions, eps):
    """x [T, heads, 128] -> (normed and turned, |a| + |b| of the turned pair), in 64 bits."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = y[..., :D // 2], y[..., D // 2:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


def attention(q, k, v, cu, positions, tables, scale):
    """q [T, Hq, 128]; k, v unpacked pools.  Returns (o, sum p |v|) [T, Hq, 128], zeros where nothing is seen."""
    q = np.asarray(q, np.float64)
    T, Hq, _ = q.shape
    P, Hkv = k.shape[:2]
    G = Hq // Hkv
    out, size = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    for b in range(len(cu) - 1):
        rows = range(int(cu[b]), int(cu[b + 1]))
        if not rows:
            continue
        last = int(positions[rows[-1]])
        n = min(-(-(last + 1) // PAGE), tables.shape[1])
        ids = np.array(tables[b, :n])
        held = (ids >= 0) & (ids < P)
        ids = np.where(held, ids, 0)
        key = np.arange(n * PAGE)
        there = np.repeat(held, PAGE) & (key <= last)
        for g in range(Hkv):
            kk = np.where(there[:, None], k[ids, g].reshape(-1, D), 0.0)
            vv = np.where(there[:, None], v[ids, g].reshape(-1, D), 0.0)
            for t in rows:
                seen = there & (key <= int(positions[t]))
                if not seen.any():
                    continue
                s = np.where(seen, scale * (q[t, g * G:(g + 1) * G] @ kk.T), -math.inf)
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[t, g * G:(g + 1) * G] = p @ vv
                size[t, g * G:(g + 1) * G] = p @ np.abs(vv)
    return out, size
