"""The 4-bit cache's operators where batches, pages and values are unusual: rows that sequences share, pages that were given back,
values of very unequal size."""
import math

import numpy as np
import pytest

from moe_infer_b200 import _lib as L

from . import kv4_ref as R
from .test_gpu_kv4 import Case, as_f64, as_type, bound_of, eng  # noqa: F401  (eng: fixture)

pytestmark = pytest.mark.gpu


# ─── batches that break their bounds ────────────────────────────────────────
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_start", [[0, 300, 0, 300, 0, 300], [0, 150, 300, 0, 300, 20, 300, 0, 300]])
def test_prompts_that_share_rows(eng, q_start, dim):  # noqa: F811
    """q_start runs back: every sequence that counts up is within n_tokens, together they have more rows than the call's work
    area was made for.  Reported; the cache, the queries and memory behind the work area keep what they hold."""
    n = len(q_start) - 1
    c = Case(eng, [320] * n, [1] * n, kv_heads=1, dim=dim, page=16, seed=3)
    c.fill()
    q = as_type(c.rng.standard_normal((300, 1, dim)), L.DT_BF16)
    qb, out = c.up(q), c.up(np.zeros_like(q))
    # the work area grows to this call's size first, then a buffer is placed behind it
    eng.kv4_attention_dev(c.cache, c.batch_of([0, 150, 300] + [300] * (n - 2), 300, 300), qb.ptr, out.ptr, L.DT_BF16, 1, scale=0.1)
    eng.sync()
    guard = c.up(np.full(1 << 22, 0xA5, np.uint8))
    before = c.pages.download(np.uint8, (c.bytes,))
    eng.kv4_attention_dev(c.cache, c.batch_of(q_start, 300, 300), qb.ptr, out.ptr, L.DT_BF16, 1, scale=0.1)
    with pytest.raises(ValueError, match="q_start or seq_lens"):
        eng.sync()
    assert np.array_equal(before, c.pages.download(np.uint8, (c.bytes,)))
    assert np.array_equal(q, qb.download(q.dtype, q.shape))
    assert np.all(guard.download(np.uint8, (1 << 22,)) == 0xA5)
    eng.kv4_attention_dev(c.cache, c.batch_of([0, 150, 300] + [300] * (n - 2), 300, 300), qb.ptr, out.ptr, L.DT_BF16, 1, scale=0.1)
    eng.sync()  # and the engine carries on
    c.free()


# ─── plain attention over a case's cache ────────────────────────────────────
def attend(eng, c, q, heads, dtype, *, scale, window=0, gate=None, batch=None):  # noqa: F811
    out = c.up(np.zeros_like(q))
    eng.kv4_attention_dev(c.cache, batch or c.batch, c.up(q).ptr, out.ptr, dtype, heads, scale=scale, window=window, gate=c.up(gate).ptr if gate is not None else 0)
    eng.sync()
    return as_f64(out.download(q.dtype, q.shape), dtype)


def store(eng, c, k, v):  # noqa: F811
    """Every position of every sequence, in one call."""
    start = np.concatenate([[0], np.cumsum(c.lens)])
    eng.kv4_append_dev(c.cache, c.batch_of(start, sum(c.lens), max(c.lens)), c.up(k).ptr, c.up(v).ptr, L.DT_F32)
    eng.sync()
    return R.codec(k), R.codec(v)


def close(got, want, size, reach, dtype, rows=slice(None)):
    bound = bound_of(dtype, want, size, reach)
    r = np.abs(got - want) / bound
    assert np.all(r[rows] <= 1), f"worst {np.max(r[rows]):.3f} of the bound"


# shapes that take every kernel: few rows (one and two columns of eight), many f32 rows, prompts of bf16 rows
FORMS = [(t, lens, q_lens) for lens, q_lens in (([300], [1]), ([300, 200], [4, 3]), ([700, 600], [700, 600])) for t in (L.DT_F32, L.DT_BF16)]


# ─── windows ────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 8, 8), (256, 16, 2)])
@pytest.mark.parametrize("lens,q_lens", [([900, 333], [1, 1]), ([900, 333], [3, 3]), ([900, 700], [550, 500])])
def test_pages_behind_the_window_may_be_gone(eng, lens, q_lens, dim, heads, kv_heads, dtype):  # noqa: F811
    """Pages that end before the first position a row sees are not looked up: their table entries may be anything (-1 here)."""
    for window in (1, 37, 130):
        c = Case(eng, lens, q_lens, kv_heads=kv_heads, dim=dim, page=16, seed=window)
        k, v = c.fill()
        for b, (n, nq) in enumerate(zip(lens, q_lens)):
            c.table[b, :max(n - nq - window + 1, 0) // 16] = -1
        q = as_type(c.rng.standard_normal((c.rows, heads, dim)), dtype)
        want, size, reach = R.attention(as_f64(q, dtype), k, v, lens, q_lens, window, 0.1)
        close(attend(eng, c, q, heads, dtype, scale=0.1, window=window, batch=c.batch_of(c.q_start, c.rows, c.max_q)), want, size, reach, dtype)
        c.free()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("lens,q_lens", [([5, 40], [9, 2]), ([90], [400]), ([600], [700])])
@pytest.mark.parametrize("window", [0x7FFFFFFF, 0x7FFFFFF0, 0x7FFE0000])
def test_widest_windows(eng, lens, q_lens, window, dtype):  # noqa: F811
    """A window wider than any sequence sees everything, for rows of a sequence that has more rows than positions too."""
    c = Case(eng, lens, q_lens, kv_heads=2, dim=64, page=16, seed=1)
    k, v = c.fill()
    q = as_type(c.rng.standard_normal((c.rows, 16, 64)), dtype)
    want, size, reach = R.attention(as_f64(q, dtype), k, v, lens, q_lens, 0, 0.1)
    batch = c.batch_of(c.q_start, c.rows, c.max_q)
    batch.max_seq_len = 0x7FFF0000  # a bound no tighter than it has to be
    close(attend(eng, c, q, 16, dtype, scale=0.1, window=window, batch=batch), want, size, reach, dtype)
    close(attend(eng, c, q, 16, dtype, scale=0.1, window=window), want, size, reach, dtype)
    c.free()


# ─── values and keys of unequal size ────────────────────────────────────────
# Bounds: bound_of, whose size is of an element's own group of 64.  What the other groups, other positions' weights and positions
# that a row does not see hold adds nothing to it.
@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("big", [2.0 ** 4, 2.0 ** 11, 1e5, 1e8, 1e30])
def test_large_values_that_rows_do_not_see(eng, big, dim, dtype, lens, q_lens):  # noqa: F811
    """Positions behind a row's own, or before its window, in the tile it reads: large values (and keys) there change nothing."""
    for window, keys in ((0, 1), (0, 0), (20, 1), (20, 0)):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=dim, page=16, seed=11)
        k, v = (c.rng.standard_normal((sum(lens), 1, dim)).astype(np.float32) for _ in range(2))
        at = 0
        hidden = np.zeros(c.rows, bool)
        hit = {n - 1 if nq > 1 else n - 25 for n, nq in zip(lens, q_lens)}
        for b, (n, nq) in enumerate(zip(lens, q_lens)):
            base, pos = sum(lens[:b]), np.arange(n - nq, n)
            p = n - 1 if nq > 1 else n - 25  # the last row's own position; or one just before the window of the only row
            v[base + p] *= big
            if keys:
                k[base + p] *= min(big, 1e15)
            hidden[at:at + nq] = (pos < p) | ((pos - p >= window) if window else False)
            at += nq
        assert hit and (hidden.any() or window == 0)
        kc, vc = store(eng, c, k, v)
        q = as_type(c.rng.standard_normal((c.rows, 8, dim)), dtype)
        got = attend(eng, c, q, 8, dtype, scale=0.1, window=window)
        with np.errstate(all="ignore"):
            want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, window, 0.1)
        close(got, want, size, reach, dtype, hidden)
        c.free()


@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("big", [2.0 ** 5, 2.0 ** 11, 2.0 ** 13, 1e5, 1e8, 1e30, 1e-3, 1e-8, 1e-30])
def test_groups_of_unequal_size(eng, big, dim, dtype, lens, q_lens):  # noqa: F811
    """One group of 64 of a head holds values `big` times the others', at all positions or at a few."""
    for every in (1, 97):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=dim, page=16, seed=12)
        k, v = (c.rng.standard_normal((sum(lens), 1, dim)).astype(np.float32) for _ in range(2))
        v[::every, :, 64:128] *= big
        kc, vc = store(eng, c, k, v)
        q = as_type(c.rng.standard_normal((c.rows, 8, dim)), dtype)
        want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, 0, 0.1)
        close(attend(eng, c, q, 8, dtype, scale=0.1), want, size, reach, dtype)
        c.free()


@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("big", [1e5, 1e9])
def test_large_values_of_small_weight(eng, big, dim, dtype, lens, q_lens):  # noqa: F811
    """Positions that a row sees, with weights of 1e-3 to 1e-12 of the largest, hold large values: in every group, and in one."""
    for part in (slice(0, dim), slice(0, 64)):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=dim, page=16, seed=13)
        k, v = (c.rng.standard_normal((sum(lens), 1, dim)).astype(np.float32) for _ in range(2))
        k[..., 0] = 0.0
        rows = np.arange(3, sum(lens), 41)
        k[rows, 0, 0] = -c.rng.uniform(1.0, 4.0, len(rows))
        v[rows, 0, part] *= big
        kc, vc = store(eng, c, k, v)
        qf = c.rng.standard_normal((c.rows, 8, dim))
        qf[..., 0] = 70.0
        q = as_type(qf, dtype)
        want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, 0, 0.1)
        close(attend(eng, c, q, 8, dtype, scale=0.1), want, size, reach, dtype)
        c.free()


@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("big", [1e3, 1e12, 1e30])
def test_values_of_zero_with_the_largest_weight(eng, big, dtype, lens, q_lens):  # noqa: F811
    """The first position takes most of the weight and holds zeros, the others hold large values."""
    for dim in (64, 256):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=dim, page=16, seed=18)
        k, v = (c.rng.standard_normal((sum(lens), 1, dim)).astype(np.float32) for _ in range(2))
        v *= np.float32(big)
        for b in range(len(lens)):
            k[sum(lens[:b]), 0, 0] = 4.0
            v[sum(lens[:b])] = 0.0
        kc, vc = store(eng, c, k, v)
        qf = c.rng.standard_normal((c.rows, 8, dim))
        qf[..., 0] = 40.0
        q = as_type(qf, dtype)
        want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, 0, 0.1)
        close(attend(eng, c, q, 8, dtype, scale=0.1), want, size, reach, dtype)
        c.free()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("small", [0.0, 1e-12, 1e-30])
def test_long_runs_of_zeros(eng, small, dtype):  # noqa: F811
    """Thousands of positions whose values are zeros (or tiny) take all of the weight, scores a little above the first ones'."""
    n, rows = 20000, 200
    c = Case(eng, [n], [rows], kv_heads=1, dim=64, page=64, seed=23)
    k, v = (0.01 * c.rng.standard_normal((n, 1, 64)).astype(np.float32) for _ in range(2))
    k[128:, 0, 0] = 1.369  # 7.9 powers of two above the first 128
    v[:n - rows] *= np.float32(small)
    k[n - rows:, 0, 0] = 0.0
    kc, vc = store(eng, c, k, v)
    qf = c.rng.standard_normal((rows, 4, 64))
    qf[..., 0] = 40.0
    q = as_type(qf, dtype)
    want, size, reach = R.attention(as_f64(q, dtype), kc, vc, [n], [rows], 0, 0.1)
    close(attend(eng, c, q, 4, dtype, scale=0.1), want, size, reach, dtype)
    c.free()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("window", [0, 90])
def test_sequences_of_unequal_and_ordinary_values_in_one_call(eng, window, dtype):  # noqa: F811
    """Prompts, verifications and single tokens, some of them over values and keys of very unequal size, gated; twice, so that
    nothing of the first call decides about the second."""
    lens, q_lens = [700, 300, 250, 90, 500, 0, 333], [700, 300, 1, 40, 350, 1, 333]
    c = Case(eng, lens, q_lens, kv_heads=2, dim=128, page=16, seed=19)
    first = np.cumsum([0] + lens)
    for unequal in ((1, 2, 3), (0, 4), ()):
        k, v = (c.rng.standard_normal((sum(lens), 2, 128)).astype(np.float32) for _ in range(2))
        for b in unequal:
            v[first[b] + 5:first[b + 1]:50, :, 64:] *= 1e7
            k[first[b] + 30:first[b + 1]:70, 1, :64] *= 1e-7
        kc, vc = store(eng, c, k, v)
        q, g = (as_type(c.rng.standard_normal((c.rows, 8, 128)), dtype) for _ in range(2))
        want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, window, 0.1)
        s = 1 / (1 + np.exp(-as_f64(g, dtype)))
        close(attend(eng, c, q, 8, dtype, scale=0.1, window=window, gate=g), want * s, size * s, reach, dtype)
    c.free()


def test_prompts_among_many_sequences(eng):  # noqa: F811
    """More sequences than a CTA has threads before a prompt, and the images of two prompts."""
    rng = np.random.default_rng(20)
    lens, q_lens = [int(x) for x in rng.integers(0, 60, 700)], [1] * 700
    for b, n in ((290, 150), (655, 70), (699, 210)):
        lens[b], q_lens[b] = n, n - 3
    c = Case(eng, lens, q_lens, kv_heads=2, dim=64, page=16, seed=20)
    k, v = c.fill()
    q = as_type(c.rng.standard_normal((c.rows, 4, 64)), L.DT_BF16)
    want, size, reach = R.attention(as_f64(q, L.DT_BF16), k, v, lens, q_lens, 0, 0.1)
    close(attend(eng, c, q, 4, L.DT_BF16, scale=0.1), want, size, reach, L.DT_BF16)
    c.free()


@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("big", [1e3, 1e5, 1e15])
def test_scores_of_any_size(eng, big, dtype, lens, q_lens):  # noqa: F811
    """Scores up to 10^31: the position with the largest one (by a thousandth of what scores are made of) is the result."""
    c = Case(eng, lens, q_lens, kv_heads=1, dim=64, page=16, seed=24)
    k, v = (c.rng.standard_normal((sum(lens), 1, 64)).astype(np.float32) for _ in range(2))
    kc, vc = store(eng, c, k * np.float32(big), v)
    q = as_type(c.rng.standard_normal((c.rows, 8, 64)) * big, dtype)
    got = attend(eng, c, q, 8, dtype, scale=0.1)
    assert np.isfinite(got).all()
    qd, at, seen = as_f64(q, dtype), 0, 0
    for b, (n, nq) in enumerate(zip(lens, q_lens)):
        kb, vb = (x[sum(lens[:b]):sum(lens[:b]) + n, 0].astype(np.float64) for x in (kc, vc))
        for h in range(8):
            s = 0.1 * qd[at:at + nq, h] @ kb.T
            s[np.arange(n)[None] > np.arange(n - nq, n)[:, None]] = -np.inf
            best = s.argmax(1)
            rest = s.copy()
            rest[np.arange(nq), best] = -np.inf
            sure = s.max(1) - rest.max(1) > 1e-3 * 0.1 * (np.abs(qd[at:at + nq, h]) @ np.abs(kb).max(0))
            err = np.abs(got[at:at + nq, h] - vb[best])[sure]
            # one weight, 1: what is left is the value's own rounding (2^-8, or 2^-19 of the group's range and |value|)
            assert np.all(err <= np.abs(vb[best])[sure] * 2.0 ** -8 + 8 * 2.0 ** (-19 if dtype == L.DT_F32 else -11))
            seen += sure.sum()
        at += nq
    assert seen > 0
    c.free()


@pytest.mark.parametrize("heads", [128, 130])
def test_many_heads_per_kv_head(eng, heads):  # noqa: F811
    """One token's query heads alone are a prompt's rows; with values that such a kernel leaves to the other."""
    lens, q_lens = [300, 200, 50, 0, 90], [1, 4, 20, 1, 90]
    for big in (1.0, 1e6):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=128, page=16, seed=25)
        k, v = (c.rng.standard_normal((sum(lens), 1, 128)).astype(np.float32) for _ in range(2))
        v[10:320:20, :, 64:] *= big
        kc, vc = store(eng, c, k, v)
        q = as_type(c.rng.standard_normal((c.rows, heads, 128)), L.DT_BF16)
        want, size, reach = R.attention(as_f64(q, L.DT_BF16), kc, vc, lens, q_lens, 0, 0.1)
        close(attend(eng, c, q, heads, L.DT_BF16, scale=0.1), want, size, reach, L.DT_BF16)
        c.free()


# A score is the sum over groups of s (q . n) and b sum(q), both of which may be larger than the sum of q_d k_d: its error is
# relative to sum |q_d| (|k_d| + 15 s), not to sum |q_d k_d| alone.  2^-24 of it for each of the (at most three) f32 roundings of
# a group's terms, 2^-23 for the 22-bit query operands, some 2^-22 for the MMA's sums: 2^-21, and a weight is off by twice that.
# bf16 rows: queries are exact, prompts hold keys to 2^-12 of |k|, which bound_of counts.
@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("big", [20.0, 300.0, 1e6])
def test_key_channels_of_unequal_size(eng, big, dim, dtype, lens, q_lens):  # noqa: F811
    """A few channels of the keys are `big` times the others (of one sign, as real caches have them), the queries small there."""
    c = Case(eng, lens, q_lens, kv_heads=1, dim=dim, page=16, seed=14)
    k, v = (c.rng.standard_normal((sum(lens), 1, dim)).astype(np.float32) for _ in range(2))
    k[..., [5, dim - 3]] = big * (1 + 0.1 * c.rng.standard_normal((sum(lens), 1, 2)))
    kc, vc = store(eng, c, k, v)
    qf = c.rng.standard_normal((c.rows, 8, dim)) / big
    qf[..., [5, dim - 3]] /= 10.0
    q = as_type(qf, dtype)
    want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, 0, 0.1)
    span = np.repeat(np.ptp(kc.reshape(len(kc), -1, 64), 2), 64, 1).max(0)  # 15 s, at most, of every channel
    formed = 0.1 * (np.abs(as_f64(q, dtype)) @ (np.abs(kc[:, 0]).max(0) + span))[..., None]
    got = attend(eng, c, q, 8, dtype, scale=0.1)
    bound = bound_of(dtype, want, size, reach) + 2.0 ** -20 * formed * size
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)
    c.free()


@pytest.mark.parametrize("dtype,lens,q_lens", FORMS)
def test_groups_of_equal_values(eng, dtype, lens, q_lens):  # noqa: F811
    """A group of 64 equal values has no range: zeros come out as zeros, others as themselves, beside small and large ones."""
    for small in (1e-6, 1.0, 1e6):
        c = Case(eng, lens, q_lens, kv_heads=1, dim=256, page=16, seed=15)
        k, v = (c.rng.standard_normal((sum(lens), 1, 256)).astype(np.float32) for _ in range(2))
        v *= np.float32(small)
        v[..., 64:128] = 0.0
        v[..., 128:192] = 0.37e-3 * small
        v[::3] = 0.0
        k[1::7, :, 128:192] = 0.0
        kc, vc = store(eng, c, k, v)
        q = as_type(c.rng.standard_normal((c.rows, 8, 256)), dtype)
        got = attend(eng, c, q, 8, dtype, scale=0.1)
        want, size, reach = R.attention(as_f64(q, dtype), kc, vc, lens, q_lens, 0, 0.1)
        close(got, want, size, reach, dtype)
        assert np.all(got[..., 64:128] == 0.0)
        c.free()


# ─── gates ──────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("lens,q_lens", [([40] * 600, [1] * 600), ([9000, 40], [1, 1]), ([700, 600], [700, 600]), ([300], [200])])
@pytest.mark.parametrize("big", [1.0, 1e30])
def test_gates_of_any_size(eng, big, lens, q_lens, dtype):  # noqa: F811
    """The gated result against the same call's without gates, times sigmoid(gate) in 64 bits; whether a sequence was one CTA's or
    several's.  f32: exp to 2 ulp (2^-22) in the numerator, half of that in the denominator, a sum and a product (2 x 2^-24), a
    quotient to 2 ulp (2^-22), the rounding of the result without gates (2^-24): below 2^-20.  bf16: two roundings of half a
    step, 2 x 2^-8, and 2^-13."""
    c = Case(eng, lens, q_lens, kv_heads=2, dim=64, page=16, seed=16)
    k, v = (c.rng.standard_normal((sum(lens), 2, 64)).astype(np.float32) for _ in range(2))
    store(eng, c, k, v * np.float32(big))
    q = as_type(c.rng.standard_normal((c.rows, 16, 64)), dtype)
    g = as_type(c.rng.uniform(-87, 87, (c.rows, 16, 64)), dtype)
    plain = attend(eng, c, q, 16, dtype, scale=0.1)
    got = attend(eng, c, q, 16, dtype, scale=0.1, gate=g)
    want = plain / (1 + np.exp(-as_f64(g, dtype)))
    assert np.isfinite(got).all() and np.abs(plain).max() > 0.1 * big
    err = np.abs(got - want) / (np.abs(want) * (2.0 ** -20 if dtype == L.DT_F32 else 2.0 ** -7 + 2.0 ** -13) + 2.0 ** -126)
    assert err.max() <= 1, err.max()
    c.free()


# ─── rotary positions outside the table ─────────────────────────────────────
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("lens,q_lens,kv_heads,dim,rotary,interleaved", [([40, 21], [19, 2], 2, 128, 64, 0), ([40, 21], [19, 2], 2, 128, 20, 1), ([40, 21], [19, 2], 1, 64, 64, 1),
                                                                         ([1813, 1502], [1810, 1502], 8, 64, 32, 1), ([1813, 1502], [1810, 1502], 6, 256, 64, 0)])
def test_append_skips_rows_without_a_rotation(eng, lens, q_lens, kv_heads, dim, rotary, interleaved, dtype):  # noqa: F811
    """A row whose position the table does not hold is reported, and neither its key nor its value is stored; the others are."""
    from moe_infer_b200.native import RopeTable, rope_table
    c = Case(eng, lens, q_lens, kv_heads=kv_heads, dim=dim, page=48, seed=17)
    k_old, v_old = c.fill()
    k, v = (as_type(c.rng.standard_normal((c.rows, kv_heads, dim)), dtype) for _ in range(2))
    tab = rope_table(rotary, 500, 1e4)
    pos = c.rng.integers(0, 500, c.rows).astype(np.int32)
    bad = c.rng.random(c.rows) < 0.2
    bad[[0, c.rows - 1]] = True
    pos[bad] = c.rng.choice([-1, 500, 1 << 30, -(1 << 31)], bad.sum())
    rope = RopeTable(c.up(tab).ptr, 500, rotary, interleaved)
    eng.kv4_append_dev(c.cache, c.batch, c.up(k).ptr, c.up(v).ptr, dtype, rope=rope, rope_positions=c.up(pos).ptr)
    with pytest.raises(ValueError, match="rotary table"):
        eng.sync()
    ko, vo = c.up(np.zeros(k.shape, np.float32)), c.up(np.zeros(k.shape, np.float32))
    eng.kv4_gather_dev(c.cache, c.batch, ko.ptr, vo.ptr, L.DT_F32)
    eng.sync()
    own = np.concatenate([np.arange(sum(lens[:b]) + n - nq, sum(lens[:b]) + n) for b, (n, nq) in enumerate(zip(lens, q_lens))])
    kf, vf = as_f64(k, dtype).astype(np.float32), as_f64(v, dtype).astype(np.float32)
    k_new = R.codec(R.rotate_f32(kf, tab[np.where(bad, 0, pos)], interleaved))
    np.testing.assert_array_equal(ko.download(np.float32, k.shape), np.where(bad[:, None, None], k_old[own], k_new))
    np.testing.assert_array_equal(vo.download(np.float32, k.shape), np.where(bad[:, None, None], v_old[own], R.codec(vf)))
    # the same for positions that follow from the cache and pass the table's end
    short = RopeTable(c.up(tab).ptr, max(lens) - 1, rotary, interleaved) if max(lens) <= 500 else None
    if short:
        eng.kv4_append_dev(c.cache, c.batch, c.up(k).ptr, c.up(v).ptr, dtype, rope=short)
        with pytest.raises(ValueError, match="rotary table"):
            eng.sync()
    c.free()


# ─── the call's work area ───────────────────────────────────────────────────
def test_capture_is_refused(eng):  # noqa: F811
    """The work area moves when it grows, so attention is not captured; the capture itself and the engine go on."""
    import ctypes
    cu = ctypes.CDLL("libcuda.so.1")
    c = Case(eng, [300], [300], kv_heads=1, dim=64, page=16, seed=21)
    k, v = c.fill()
    stream, graph = ctypes.c_void_p(eng.stream()), ctypes.c_void_p()
    for dtype in (L.DT_F32, L.DT_BF16):
        q = as_type(c.rng.standard_normal((c.rows, 4, 64)), dtype)
        qb, out = c.up(q), c.up(np.zeros_like(q))
        assert cu.cuStreamBeginCapture_v2(stream, 2) == 0
        with pytest.raises(L.MoeError, match="captured"):
            eng.kv4_attention_dev(c.cache, c.batch, qb.ptr, out.ptr, dtype, 4, scale=0.1)
        assert cu.cuStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert cu.cuGraphDestroy(graph) == 0
        want, size, reach = R.attention(as_f64(q, dtype), k, v, [300], [300], 0, 0.1)
        close(attend(eng, c, q, 4, dtype, scale=0.1), want, size, reach, dtype)
    c.free()


def test_work_area_grows_in_steps(native_lib):
    """A prompt in chunks: each call may need a little more than the one before, and few of them allocate."""
    import ctypes
    from moe_infer_b200.native import Dims, NativeEngine
    cu, free, total = ctypes.CDLL("libcuda.so.1"), ctypes.c_size_t(), ctypes.c_size_t()
    e = NativeEngine(Dims(num_experts=4, top_k=4, num_layers=1))
    n = 64 * 128
    c = Case(e, [n], [128], kv_heads=8, dim=256, page=16, seed=22)
    c.fill()
    q = c.up(as_type(c.rng.standard_normal((128, 8, 256)), L.DT_BF16))
    out = c.up(np.zeros((128, 8, 256), np.uint16))
    changes, last = 0, None
    for chunk in range(1, 65):
        e.kv4_attention_dev(c.cache, c.batch_of([0, 128], 128, 128, [128 * chunk]), q.ptr, out.ptr, L.DT_BF16, 8, scale=0.1)
        e.sync()
        c.keep.pop().free(), c.keep.pop().free(), c.keep.pop().free()  # the batch's arrays
        assert cu.cuMemGetInfo_v2(ctypes.byref(free), ctypes.byref(total)) == 0
        changes += last is not None and abs(free.value - last) >= 1 << 20
        last = free.value
    # from 1 tile to 64 by a factor of 1.5 each: 11 steps
    assert changes <= 12, changes
    c.free()
    e.close()
