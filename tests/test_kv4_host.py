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


GOOD = dict(cache=(1 << 20, 8, 16, 2, 128), batch=(1 << 20, 1 << 20, 1 << 20, 2, 6, 4, 60, 3), rope=(1 << 20, 100, 32, 0))


def call(lib, which, *, cache=GOOD["cache"], batch=GOOD["batch"], rope=GOOD["rope"], x=1 << 21, y=1 << 22, z=1 << 23, strides=None, dtype=0, heads=8,
         scale=0.1, window=0, positions=1 << 20, dim=128, tokens=6):
    """An entry point without an engine: whatever is wrong with the arguments is said first."""
    c, b = Kv4Cache(*cache), Kv4Batch(*batch)
    r = RopeTable(*rope) if rope else None
    kv = cache[3] * cache[4]
    if which == "rope":
        xs, os_ = strides or ((heads * dim, dim), (heads * dim, dim))
        st = lib.moe_rope_dev(None, r, x, *xs, y, *os_, dtype, tokens, heads, dim, positions)
    elif which == "append":
        xs, os_ = strides or ((kv, cache[4]), (kv, cache[4]))
        st = lib.moe_kv4_append_dev(None, c, b, x, *xs, y, *os_, dtype, r, positions)
    elif which == "gather":
        st = lib.moe_kv4_gather_dev(None, c, b, x, y, dtype)
    else:
        xs, os_ = strides or ((heads * cache[4], cache[4]), (heads * cache[4], cache[4]))
        st = lib.moe_kv4_attention_dev(None, c, b, x, *xs, z, *os_, y, dtype, heads, scale, window)
    assert st == L.ERR_INVALID
    return L.last_error()


def test_null_engine_is_refused(native_lib):
    for which in ("rope", "append", "gather", "attention"):
        assert "null engine" in call(native_lib, which)
    assert native_lib.moe_engine_stream(None, C.byref(C.c_void_p())) == L.ERR_INVALID


CACHE, BATCH, ROPE = GOOD["cache"], GOOD["batch"], GOOD["rope"]


def but(t, i, v):
    return t[:i] + (v,) + t[i + 1:]


@pytest.mark.parametrize("kw,says", [
    (dict(cache=but(CACHE, 4, 96)), "head_dim"), (dict(cache=but(CACHE, 2, 24)), "page_size"), (dict(cache=but(CACHE, 2, 0)), "page_size"),
    (dict(cache=but(CACHE, 3, 0)), "num_kv_heads"), (dict(cache=but(CACHE, 0, None)), "null pages"), (dict(cache=but(CACHE, 0, (1 << 20) + 8)), "aligned"),
    (dict(cache=but(CACHE, 1, -1)), "num_pages"), (dict(batch=but(BATCH, 0, None)), "q_start"), (dict(batch=but(BATCH, 1, None)), "seq_lens"),
    (dict(batch=but(BATCH, 2, None)), "page_table"), (dict(batch=but(BATCH, 3, -1)), "negative"), (dict(batch=but(BATCH, 4, -1)), "negative"),
    (dict(batch=but(BATCH, 6, -1)), "negative"), (dict(batch=but(BATCH, 6, 0x7FFFFFFF)), "max_seq_len"), (dict(dtype=2), "f32 or bf16"),
    (dict(x=None), "null argument"), (dict(y=None), "null argument"), (dict(x=(1 << 21) + 1), "misaligned")])
@pytest.mark.parametrize("which", ["append", "gather", "attention"])
def test_cache_refusals(native_lib, which, kw, says):
    assert says in call(native_lib, which, **kw)


def test_append_and_gather_refusals(native_lib):
    assert "rotary_dim" in call(native_lib, "append", rope=but(ROPE, 2, 160))
    assert "rotary_dim" in call(native_lib, "append", rope=but(ROPE, 2, 31))
    assert "no positions" in call(native_lib, "append", rope=but(ROPE, 1, 0))
    assert "null table" in call(native_lib, "append", rope=but(ROPE, 0, None))
    assert "without a rope table" in call(native_lib, "append", rope=None)
    assert "negative stride" in call(native_lib, "append", strides=((-1, 128), (256, 128)))
    assert "overlap" in call(native_lib, "gather", y=(1 << 21) + 64)


def test_attention_refusals(native_lib):
    assert "num_heads" in call(native_lib, "attention", heads=7)
    assert "num_heads" in call(native_lib, "attention", heads=0)
    assert "window" in call(native_lib, "attention", window=-1)
    assert "finite" in call(native_lib, "attention", scale=float("nan"))
    assert "finite" in call(native_lib, "attention", scale=float("inf"))
    assert "negative stride" in call(native_lib, "attention", strides=((1024, -128), (1024, 128)))
    assert "16-byte" in call(native_lib, "attention", y=(1 << 22) + 4)
    assert "overlaps" in call(native_lib, "attention", y=1 << 21)
    assert "overlaps" in call(native_lib, "attention", y=(1 << 23) + 1024)


def test_rope_refusals(native_lib):
    assert "rotary_dim" in call(native_lib, "rope", rope=but(ROPE, 2, 130))
    assert "bad shape" in call(native_lib, "rope", heads=0)
    assert "bad shape" in call(native_lib, "rope", tokens=-1)
    assert "f32 or bf16" in call(native_lib, "rope", dtype=3)
    assert "null argument" in call(native_lib, "rope", positions=None)
    assert "misaligned" in call(native_lib, "rope", y=(1 << 22) + 2)
    assert "overlap" in call(native_lib, "rope", strides=((1024, 128), (128, 128)))          # output rows overlap
    assert "in place" in call(native_lib, "rope", y=1 << 21, strides=((2048, 256), (1024, 128)))
    assert "without being the same" in call(native_lib, "rope", y=(1 << 21) + 4096)
    assert "negative stride" in call(native_lib, "rope", strides=((-1, 128), (1024, 128)))
    # heads outermost is fine: the next thing missing is the engine
    assert "null engine" in call(native_lib, "rope", strides=((1024, 128), (128, 768)))


def test_empty_batches_need_nothing(native_lib):
    for batch in (but(BATCH, 3, 0), but(BATCH, 4, 0), but(BATCH, 7, 0)):
        c, b = Kv4Cache(*CACHE), Kv4Batch(*batch)
        assert native_lib.moe_kv4_append_dev(None, c, b, None, 1, 1, None, 1, 1, 0, None, None) == L.MOE_OK
        assert native_lib.moe_kv4_gather_dev(None, c, b, None, None, 0) == L.MOE_OK
        assert native_lib.moe_kv4_attention_dev(None, c, b, None, 1, 1, None, 0, 0, None, 0, 8, 1.0, 0) == L.MOE_OK
