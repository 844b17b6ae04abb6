"""The oracle of the 8-bit paged KV cache (oracle/kv8_oracle.py) against torch's own e4m3 conversion, closed forms
and brute force, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv8_oracle as kv


def test_e4m3_round_trip_and_ties():
    codes = np.arange(256, dtype=np.uint8)
    ref = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv.from_e4m3(codes), ref, equal_nan=True)
    v = kv.e4m3_values()
    ties = np.concatenate([(v[1:] + v[:-1]) / 2, np.nextafter(v[1:], 0), v, np.linspace(0, 448, 9999)])
    ties = np.concatenate([ties, -ties]).astype(np.float32)
    ref = torch.from_numpy(ties).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kv.to_e4m3(ties), ref)
    assert list(kv.to_e4m3([1e9, -np.inf, np.nan])) == [0x7E, 0xFE, 0x7F]


def test_scale_is_the_smallest_power_of_two():
    assert kv.scale_of(448.0) == 1.0 and kv.scale_of(np.nextafter(448.0, 1e9)) == 2.0
    assert kv.scale_of(0.0) == 2.0 ** -100 and kv.scale_of(3.5) == 2.0 ** -7
    for a in np.exp(np.random.default_rng(0).uniform(-30, 30, 200)):
        s = kv.scale_of(a)
        assert a / s <= 448 < 2 * a / s


@pytest.mark.parametrize("index,shape", [(kv.k_index, (8, 16, 16)), (kv.v_index, (2, 4, 64, 4))])
def test_append_and_unpack(index, shape):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((21, 2, 128))
    codes, scale = rng.integers(0, 120, (3, 2, *shape)).astype(np.uint8), np.full((3, 2), 2.0 ** -6)
    slots = np.concatenate([np.arange(2 * 16 + 13, 2 * 16 + 16), np.arange(16), [-1, 16 * 3]])  # page 2 goes on, page 0 begins
    before = kv.unpack(codes, scale, index)
    kv.append(x, slots, None, codes, scale, index)
    after = kv.unpack(codes, scale, index)
    assert np.array_equal(after[1], before[1])
    # a code is off by half a step: 2^-4 of a normal value, 2^-10 scales of a subnormal
    assert (np.abs(after[2][:, 13:] - x[:3].transpose(1, 0, 2)) <= 2.0 ** -4 * np.abs(x[:3].transpose(1, 0, 2)) + 2.0 ** -10 *
            scale[2][:, None, None]).all()
    assert (np.abs(after[2][:, :13] - before[2][:, :13]) <= 2.0 ** -10 * scale[2][:, None, None]).all()
    assert (np.abs(after[0] - x[3:19].transpose(1, 0, 2)) <= 2.0 ** -4 * np.abs(x[3:19].transpose(1, 0, 2)) + 2.0 ** -10 *
            scale[0][:, None, None]).all()


def test_plan_by_hand():
    tables = np.full((4, 3), -7, np.int32)
    tables[0, :1], tables[2, :2] = 4, (9, 8)
    pos, slot, cu, ctx, out, used = kv.plan([15, 0, 20, 40], [3, 0, 1, 30], tables, [5, 6], 12, 8)
    assert list(cu) == [0, 3, 3, 4, 12] and list(ctx) == [18, 0, 21, 48] and used == 1
    assert list(pos[:4]) == [15, 16, 17, 20] and list(slot[:4]) == [4 * 16 + 15, 5 * 16, 5 * 16 + 1, 8 * 16 + 4]
    assert out[0].tolist() == [4, 5, -7] and out[2].tolist() == [9, 8, -7] and out[3].tolist() == [-7] * 3
    assert (slot[4:] == -1).all() and list(pos[4:]) == list(range(40, 48))


def test_attention_of_equal_keys_is_the_mean():
    rng = np.random.default_rng(2)
    k, v = np.ones((4, 1, 16, 128)), rng.standard_normal((4, 1, 16, 128))
    tables = np.array([[2, -1, 0]], np.int32)
    o, size = kv.attention(rng.standard_normal((2, 3, 128)), k, v, [0, 2], [35, 36], tables, 0.1)
    seen = np.concatenate([v[2, 0], v[0, 0, :5]])
    assert np.allclose(o[1], seen.mean(0)) and np.allclose(size[1], np.abs(seen).mean(0))
    assert np.allclose(o[0], np.concatenate([v[2, 0], v[0, 0, :4]]).mean(0))


def test_rotary_keeps_pairs_norms():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3, 2, 128))
    y, _ = kv.norm_rope(x, np.ones(128), 1e6 ** (-np.arange(0, 128, 2) / 128), [0, 7, 100000], 0.0)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True))
    assert np.allclose(y[0], n[0])
    assert np.allclose(y[..., :64] ** 2 + y[..., 64:] ** 2, n[..., :64] ** 2 + n[..., 64:] ** 2)
