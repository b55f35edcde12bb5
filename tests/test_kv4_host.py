"""Rotary tables and the refusals of the rotary and 4-bit cache entry points (no GPU needed)."""
import ctypes as C
import math

import numpy as np
import pytest

from moe_infer_b200 import _lib as L
from moe_infer_b200.native import Kv4Batch, Kv4Cache, RopeTable, kv4_page_bytes, rope_table


def angles(rotary, theta, n, *, factor=None, ramp=None, first=0):
    freq = theta ** (-2.0 * np.arange(rotary // 2) / rotary)
    if factor is not None:
        w = np.ones(rotary // 2) if ramp is None else ramp
        freq = freq / factor * w + freq * (1 - w)
    return np.arange(first, first + n)[:, None] * freq


def check_table(got, a, mul=1.0):
    # one rounding to f32 (half a step, of values of at most mul), and the last bits of a 64-bit angle of some 10^5
    want = np.concatenate([np.cos(a), np.sin(a)], 1) * mul
    assert got.dtype == np.float32 and got.shape == want.shape
    assert np.max(np.abs(got - want)) <= 2.0 ** -24 * mul + 1e-9


def test_rope_tables(native_lib):
    check_table(rope_table(64, 300, 1e7), angles(64, 1e7, 300))
    check_table(rope_table(2, 10, 1e4, first_position=200000), angles(2, 1e4, 10, first=200000))
    check_table(rope_table(128, 50, 1e4, scaling=L.ROPE_LINEAR, factor=8.0, first_position=100000), angles(128, 1e4, 50, factor=8.0, first=100000))
    check_table(rope_table(64, 50, 1e4, scaling=L.ROPE_NTK, factor=4.0), angles(64, 1e4 * 4.0 ** (64 / 62), 50))
    edge = [64 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(1e4)) for t in (32.0, 1.0)]
    low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), 63)
    ramp = np.clip((np.arange(32) - low) / (high - low), 0, 1)
    assert 0 < ramp.sum() < 32
    check_table(rope_table(64, 50, 1e4, scaling=L.ROPE_YARN, factor=4.0, original_positions=4096, first_position=9000),
                angles(64, 1e4, 50, factor=4.0, ramp=ramp, first=9000), 0.1 * math.log(4.0) + 1.0)
    # frequencies that turn often keep their angle, slow ones are stretched by the factor
    assert ramp[0] == 0 and ramp[-1] == 1
    assert rope_table(64, 0, 1e4).shape == (0, 64)


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(theta=1.0), dict(theta=float("nan")), dict(scaling=7), dict(scaling=-1),
                                dict(scaling=L.ROPE_LINEAR, factor=0.5), dict(scaling=L.ROPE_YARN, factor=2.0, original_positions=0),
                                dict(scaling=L.ROPE_YARN, factor=2.0, original_positions=10, beta_fast=1.0, beta_slow=2.0),
                                dict(scaling=L.ROPE_NTK, factor=2.0, rotary_dim=2), dict(first_position=-1)])
def test_rope_table_refusals(native_lib, kw):
    args = dict(rotary_dim=64, n_positions=4, theta=1e4)
    args.update(kw)
    with pytest.raises(ValueError):
        rope_table(args.pop("rotary_dim"), args.pop("n_positions"), args.pop("theta"), **args)


def test_page_bytes(native_lib):
    # 18 bytes per 16 elements of K and V together
    assert kv4_page_bytes(16, 1, 64) == 16 * 64 * 18 // 16
    assert kv4_page_bytes(64, 2, 256) == 64 * 2 * 256 * 18 // 16
    for bad in ((15, 1, 64), (0, 1, 64), (16, 0, 64), (16, 1, 96), (-16, 1, 64)):
        with pytest.raises(ValueError):
            kv4_page_bytes(*bad)


def test_null_engine_is_refused(native_lib):
    cache, batch, rope = Kv4Cache(16, 1, 16, 1, 64), Kv4Batch(16, 16, 16, 1, 1, 1, 1, 1), RopeTable(16, 1, 8, 0)
    for st in (native_lib.moe_rope_dev(None, rope, 16, 64, 64, 16, 64, 64, 0, 1, 1, 64, 16),
               native_lib.moe_kv4_append_dev(None, cache, batch, 16, 64, 64, 16, 64, 64, 0, rope, None),
               native_lib.moe_kv4_gather_dev(None, cache, batch, 16, 16, 0),
               native_lib.moe_kv4_attention_dev(None, cache, batch, 16, 64, 64, None, 0, 0, 16, 0, 1, 1.0, 0),
               native_lib.moe_engine_stream(None, C.byref(C.c_void_p()))):
        assert st == L.ERR_INVALID
        assert "null" in L.last_error()
