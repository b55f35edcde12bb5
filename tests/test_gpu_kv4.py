"""Paged 4-bit KV cache, rotary positions and attention over the cache against plain 64-bit implementations."""
import math

import numpy as np
import pytest

from moe_infer_b200 import _lib as L
from moe_infer_b200.native import Dims, Kv4Batch, Kv4Cache, NativeEngine, RopeTable, kv4_page_bytes, rope_table

from . import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(native_lib):
    e = NativeEngine(Dims(num_experts=4, top_k=4, num_layers=1))
    yield e
    e.close()


class Case:
    """A cache in device memory with its batch: sequences of lens positions whose last q_lens are the call's rows."""

    def __init__(self, eng, lens, q_lens, *, kv_heads, dim, page, seed=0, spare_rows=0, max_q=None):
        rng = np.random.default_rng(seed)
        self.eng, self.rng, self.lens, self.q_lens = eng, rng, list(lens), list(q_lens)
        self.kv_heads, self.dim, self.page = kv_heads, dim, page
        need = [-(-n // page) for n in lens]
        self.num_pages = sum(need) + 2
        order = rng.permutation(self.num_pages)
        self.table = np.full((len(lens), max(need + [1])), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.q_start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.rows = int(self.q_start[-1])
        self.n_tokens = self.rows + spare_rows
        self.bytes = self.num_pages * kv4_page_bytes(page, kv_heads, dim)
        self.keep = []
        self.pages = self.up(rng.integers(0, 256, self.bytes, np.uint8))  # stale bytes, NaN scales among them
        self.cache = Kv4Cache(self.pages.ptr, self.num_pages, page, kv_heads, dim)
        self.max_q = max_q or max(list(q_lens) + [1])
        self.batch = self.batch_of(self.q_start, self.n_tokens, self.max_q)

    def up(self, a):
        a = np.ascontiguousarray(a)
        buf = self.eng.alloc(max(a.nbytes, 16)).upload(a)
        self.keep.append(buf)
        return buf

    def batch_of(self, q_start, n_tokens, max_q, lens=None):
        lens = self.lens if lens is None else lens
        return Kv4Batch(self.up(np.asarray(q_start, np.int32)).ptr, self.up(np.asarray(lens, np.int32)).ptr, self.up(self.table).ptr, len(lens),
                        n_tokens, self.table.shape[1], max(lens + [0]), max_q)

    def fill(self):
        """Appends every position of every sequence (in one call) and returns the values the cache then stands for."""
        total = sum(self.lens)
        k = self.rng.standard_normal((total, self.kv_heads, self.dim)).astype(np.float32)
        k *= np.exp(0.4 * self.rng.standard_normal((1, self.kv_heads, self.dim))).astype(np.float32)
        v = self.rng.standard_normal(k.shape).astype(np.float32)
        if total:
            start = np.concatenate([[0], np.cumsum(self.lens)])
            self.eng.kv4_append_dev(self.cache, self.batch_of(start, total, max(self.lens)), self.up(k).ptr, self.up(v).ptr, L.DT_F32)
            self.eng.sync()
        return R.codec(k), R.codec(v)

    def free(self):
        for b in self.keep:
            b.free()


def as_type(x, dtype):
    return x.astype(np.float32) if dtype == L.DT_F32 else R.to_bf16(x)


def as_f64(x, dtype):
    return x.astype(np.float64) if dtype == L.DT_F32 else R.from_bf16(x).astype(np.float64)


# A result may be off by what its weights are off and by its own rounding.  v = s n + b (or b + 15 s - s (15 - n)), and the two
# parts are summed apart: the first with the weights as MMA operands, the second with the weights before that rounding.  An
# error of a weight as an operand is therefore relative to at most 15 s, less than twice 8 s, any other error of a weight to |v|:
# both are covered by the weighted sum of |v| + 8 s ("size"), the first counted twice; a group holds a 0 and a 15, so 8 s is
# 8 / 15 of its range.
# A weight is off by twice (numerator and sum) the error of its score: operands of 22 bits (half a step 2^-23) and f32
# roundings of the sums over groups, which the nibbles (s n is at most a group's range) keep within a few times
# scale * sum |q k| ("reach"): 2^-22 of it in all for f32 rows, hence 2^-21 reach; then the 2-ulp exponential, the weight as
# an operand and the sums of the value pass, whose products an MMA cuts some 2^-22 below its largest, with both signs: 2^-19 for
# f32 rows (22-bit weights); 2^-11 and 2^-12 for bf16 rows (11-bit weights: half a step 2^-12, counted twice, the numerator
# against the unrounded sum), and half a step of bf16, 2^-8 of its value at most, for their result.
# Prompts of bf16 rows also hold keys and values as f16 (11 bits: half a step 2^-12 of a value, and of a key's elements, so
# 2^-12 reach in a score, twice that in a weight).
def bound_of(dtype, want, size, reach):
    if dtype == L.DT_F32:
        return size * 2.0 ** -19 + 2.0 ** -21 * reach * size + 2.0 ** -24 * np.abs(want) + 1e-30
    return size * (2.0 ** -11 + 2.0 ** -12) + 2.0 ** -11 * reach * size + 2.0 ** -8 * np.abs(want) + 1e-30


def check_attention(eng, lens, q_lens, *, heads, kv_heads, dim, page, dtype, window=0, gate=False, seed=0, spare_rows=0, q_scale=1.5, max_q=None,
                    strided=False, odd=0, scale=None):
    c = Case(eng, lens, q_lens, kv_heads=kv_heads, dim=dim, page=page, seed=seed, spare_rows=spare_rows, max_q=max_q)
    k, v = c.fill()
    wide = 2 if strided else 1
    scale = 1 / math.sqrt(dim) if scale is None else scale
    q = as_type(q_scale * c.rng.standard_normal((c.n_tokens, heads, wide * dim)), dtype)
    g = as_type(c.rng.standard_normal((c.n_tokens, heads, dim)), dtype) if gate else None
    out = c.up(np.full((c.n_tokens, heads, dim), 7, q.dtype))
    args = dict(scale=scale, window=window, q_strides=(heads * wide * dim, wide * dim))
    at = lambda x: c.up(np.concatenate([np.zeros(odd, x.dtype), x.reshape(-1)])).ptr + odd * x.dtype.itemsize  # noqa: E731  (off its alignment)
    if gate:
        args["gate"] = at(g)
    eng.kv4_attention_dev(c.cache, c.batch, at(q), out.ptr, dtype, heads, **args)
    eng.sync()
    got = out.download(q.dtype, (c.n_tokens, heads, dim))
    want, size, reach = R.attention(as_f64(q[..., :dim], dtype), k, v, lens, q_lens, window, scale)
    if gate:
        s = 1 / (1 + np.exp(-as_f64(g, dtype)[:c.rows]))
        want, size = want * s, size * s
    err = np.abs(as_f64(got[:c.rows], dtype) - want)
    bound = bound_of(dtype, want, size, reach)
    assert np.all(err <= bound), f"worst {np.max(err / bound):.3f} of the bound at {np.unravel_index(np.argmax(err / bound), err.shape)}"
    assert np.all(got[c.rows:] == np.full((), 7, q.dtype)), "rows behind the last sequence were written"
    c.free()


SHAPES = [  # heads, kv_heads, dim, page
    (16, 2, 256, 16), (4, 4, 64, 48), (8, 1, 128, 32), (14, 2, 64, 16), (24, 2, 128, 64), (5, 1, 256, 128)]


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_decode(eng, heads, kv_heads, dim, page, dtype):
    """One row per sequence; lengths of one, tile and page borders, an idle slot (a row without a position)."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 129, 255, 256, 257, 700]
    check_attention(eng, lens, [1] * len(lens), heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, spare_rows=2)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("q_len", [2, 3, 4, 7])
def test_few_rows(eng, q_len, dtype):
    lens = [40, 9, q_len, 300, 1000]
    check_attention(eng, lens, [q_len] * 5, heads=8, kv_heads=2, dim=128, page=16, dtype=dtype, gate=True)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 6, 6), (256, 16, 2)])
def test_prompts(eng, dim, heads, kv_heads, dtype):
    """Whole prompts, chunks behind a prefix, a sequence without rows, one with more rows than positions."""
    check_attention(eng, [130, 97, 50, 3, 400], [130, 33, 0, 9, 257], heads=heads, kv_heads=kv_heads, dim=dim, page=32, dtype=dtype, gate=True,
                    spare_rows=3)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_fill_the_gpu(eng, dim, dtype):
    """Enough rows for a CTA of its own per row tile."""
    check_attention(eng, [700, 900], [700, 513], heads=16, kv_heads=2, dim=dim, page=64, dtype=dtype)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("window", [1, 5, 64, 100])
def test_window(eng, window, dtype):
    check_attention(eng, [300, 64, 130], [40, 1, 130], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, window=window)
    check_attention(eng, [300, 1, 130, 500], [1] * 4, heads=16, kv_heads=2, dim=256, page=16, dtype=dtype, window=window)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_long_and_ragged(eng, dtype):
    """Units split over many CTAs next to short ones; query rows strided (head, gate)."""
    check_attention(eng, [20011, 3, 511, 9000], [1, 1, 1, 1], heads=16, kv_heads=2, dim=256, page=64, dtype=dtype, strided=True)
    check_attention(eng, [9000, 64, 2000], [2, 2, 1], heads=16, kv_heads=4, dim=128, page=16, dtype=dtype)


@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e-6, 40.0])
def test_query_sizes(eng, q_scale):
    """All-equal weights, scores that underflow to equal, and nearly one-hot weights."""
    check_attention(eng, [200, 70], [1, 1], heads=4, kv_heads=1, dim=128, page=16, dtype=L.DT_F32 if q_scale < 10 else L.DT_BF16, q_scale=q_scale)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_scales(eng, scale, dtype):
    check_attention(eng, [200, 140], [1, 130], heads=4, kv_heads=1, dim=64, page=16, dtype=dtype, scale=scale)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 14, 2), (128, 8, 8), (256, 16, 2)])
@pytest.mark.parametrize("window", [0, 1, 90, 300])
def test_batches_of_prompts_and_decodes(eng, dim, heads, kv_heads, window):
    """Prompts, chunks, verifications, single tokens, idle slots and sequences without rows in one call; rows and gates off
    their 16-byte alignment."""
    check_attention(eng, [700, 33, 1, 0, 650, 500, 64, 40], [200, 1, 1, 1, 650, 4, 0, 40], heads=heads, kv_heads=kv_heads, dim=dim, page=16,
                    dtype=L.DT_BF16, window=window, gate=True, spare_rows=1, odd=3)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("lens,q_lens", [([90], [1]), ([90], [40]), ([500, 60, 7], [2, 1, 7]), ([300, 20], [200, 20]), ([50, 400], [200, 1])])
def test_bounds_that_are_not_tight(eng, lens, q_lens, dtype):
    """max_q_len and n_tokens only bound what q_start holds: few rows where the bounds allow many, more rows than positions."""
    check_attention(eng, lens, q_lens, heads=8, kv_heads=2, dim=128, page=16, dtype=dtype, gate=True, max_q=400, spare_rows=400)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("rows", [1, 300])
def test_non_finite_queries(eng, rows, dtype):
    """A query row with a NaN or an infinity makes its own result NaN and no other."""
    c = Case(eng, [320], [rows], kv_heads=1, dim=64, page=16, seed=6)
    k, v = c.fill()
    qf = c.rng.standard_normal((rows, 4, 64)).astype(np.float32)
    bad = np.zeros((rows, 4), bool)
    for row, head, val in ((0, 1, np.nan), (rows // 2, 3, np.inf), (rows - 1, 2, -np.inf)):
        qf[row, head, 7] = val
        bad[row, head] = True
    u = np.ascontiguousarray(qf).view(np.uint32)
    q = qf if dtype == L.DT_F32 else np.where(np.isnan(qf), 0x7FC0, np.where(np.isinf(qf), u >> 16, R.to_bf16(np.where(np.isfinite(qf), qf, 0)))).astype(np.uint16)
    out = c.up(np.zeros_like(q))
    eng.kv4_attention_dev(c.cache, c.batch, c.up(q).ptr, out.ptr, dtype, 4, scale=0.125)
    eng.sync()
    got = as_f64(out.download(q.dtype, q.shape), dtype)
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    clean = np.where(bad[..., None], 0.0, as_f64(q, dtype))
    want, size, reach = R.attention(clean, k, v, [320], [rows], 0, 0.125)
    assert np.all(np.abs(got - want)[~bad] <= bound_of(dtype, want, size, reach)[~bad])
    c.free()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_unaligned_rows(eng, dtype):
    check_attention(eng, [90, 17], [2, 2], heads=8, kv_heads=2, dim=128, page=16, dtype=dtype, gate=True, odd=1)


def test_same_call_same_bits(eng):
    for dtype, q_lens in ((L.DT_F32, [1, 1]), (L.DT_BF16, [300, 7])):
        c = Case(eng, [5000, 900], q_lens, kv_heads=2, dim=128, page=16, seed=8)
        c.fill()
        q = c.up(as_type(c.rng.standard_normal((c.n_tokens, 8, 128)), dtype))
        got = []
        for _ in range(3):
            out = c.up(np.zeros((c.n_tokens, 8, 128), np.float32 if dtype == L.DT_F32 else np.uint16))
            eng.kv4_attention_dev(c.cache, c.batch, q.ptr, out.ptr, dtype, 8, scale=0.1)
            eng.sync()
            got.append(out.download(np.uint8, (c.n_tokens * 8 * 128 * (4 if dtype == L.DT_F32 else 2),)))
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
        c.free()


def test_calls_behind_one_another(eng):
    """Calls of different shapes enqueued without waiting share the engine's work area in turn."""
    cases, outs = [], []
    for k, (lens, q_lens, dtype) in enumerate((([3000], [1], L.DT_F32), ([400], [400], L.DT_BF16), ([2500, 300], [1, 1], L.DT_BF16), ([130], [130], L.DT_F32))):
        c = Case(eng, lens, q_lens, kv_heads=2, dim=128, page=16, seed=30 + k)
        kv = c.fill()
        q = as_type(c.rng.standard_normal((c.n_tokens, 8, 128)), dtype)
        outs.append((c.up(q).ptr, c.up(np.zeros_like(q)), q, kv, dtype))
        cases.append(c)
    for _ in range(2):
        for c, (qp, out, _, _, dtype) in zip(cases, outs):
            eng.kv4_attention_dev(c.cache, c.batch, qp, out.ptr, dtype, 8, scale=0.1)
    eng.sync()
    for c, (_, out, q, (k, v), dtype) in zip(cases, outs):
        want, size, reach = R.attention(as_f64(q, dtype), k, v, c.lens, c.q_lens, 0, 0.1)
        assert np.all(np.abs(as_f64(out.download(q.dtype, q.shape), dtype) - want) <= bound_of(dtype, want, size, reach))
        c.free()


def test_pages_beyond_4_gib(eng):
    """Byte offsets of pages pass 32 bits."""
    kv_heads, dim, page = 8, 256, 64
    per = kv4_page_bytes(page, kv_heads, dim)
    num = (9 << 29) // per  # 4.5 GiB
    pages = eng.alloc(num * per)
    c = Case(eng, [150, 70], [150, 1], kv_heads=kv_heads, dim=dim, page=page, seed=12)
    c.cache = Kv4Cache(pages.ptr, num, page, kv_heads, dim)
    c.table = np.array([[num - 1, 3, num - 7], [num - 2, num // 2, -1]], np.int32)
    c.batch = c.batch_of(c.q_start, c.n_tokens, c.max_q)
    k, v = c.fill()
    for dtype in (L.DT_F32, L.DT_BF16):
        q = as_type(c.rng.standard_normal((c.n_tokens, 8, dim)), dtype)
        out = c.up(np.zeros_like(q))
        eng.kv4_attention_dev(c.cache, c.batch, c.up(q).ptr, out.ptr, dtype, 8, scale=0.1)
        eng.sync()
        want, size, reach = R.attention(as_f64(q, dtype), k, v, c.lens, c.q_lens, 0, 0.1)
        assert np.all(np.abs(as_f64(out.download(q.dtype, q.shape), dtype) - want) <= bound_of(dtype, want, size, reach))
    pages.free()
    c.free()


def test_many_sequences(eng):
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 90, 333)]
    check_attention(eng, lens, [1] * len(lens), heads=4, kv_heads=2, dim=64, page=16, dtype=L.DT_BF16)


# ─── append and gather ──────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 0, 0), (64, 64, 0), (128, 32, 1), (128, 20, 0), (256, 64, 0), (256, 6, 1), (256, 256, 1)])
def test_append_is_the_codec(eng, dim, rotary, interleaved, dtype):
    """Bit for bit the rotation in f32 steps and the packer's codec, appended in several calls that begin and end inside
    quads, blocks and pages; rows behind the last sequence and other positions keep their bytes."""
    c = Case(eng, [70, 5, 33, 0], [13, 5, 1, 1], kv_heads=3, dim=dim, page=16, seed=dim + rotary, spare_rows=2)
    total = {b: c.lens[b] for b in range(4)}
    k_want = {b: np.zeros((n, 3, dim), np.float32) for b, n in total.items()}
    v_want = {b: np.zeros((n, 3, dim), np.float32) for b, n in total.items()}
    done = {b: 0 for b in total}
    tab = rope_table(rotary, 128, 1e4) if rotary else None
    rope = RopeTable(c.up(tab).ptr, 128, rotary, interleaved) if rotary else None
    for step in (1, 2, 6, 3, 29, 60):
        q = [min(step, total[b] - done[b]) for b in total]
        for b in total:
            done[b] += q[b]
        rows = sum(q)
        if rows == 0:
            continue
        k = as_type(c.rng.standard_normal((rows + 2, 3, dim)) * 3, dtype)
        v = as_type(c.rng.standard_normal((rows + 2, 3, dim)), dtype)
        batch = c.batch_of(np.concatenate([[0], np.cumsum(q)]), rows + 2, max(q), [done[b] for b in total])
        eng.kv4_append_dev(c.cache, batch, c.up(k).ptr, c.up(v).ptr, dtype, rope=rope)
        eng.sync()
        at = 0
        for b in total:
            pos = np.arange(done[b] - q[b], done[b])
            kb = as_f64(k[at:at + q[b]], dtype).astype(np.float32)
            if rotary:
                kb = R.rotate_f32(kb, tab[pos], interleaved)
            k_want[b][pos] = R.codec(kb)
            v_want[b][pos] = R.codec(as_f64(v[at:at + q[b]], dtype).astype(np.float32))
            at += q[b]
    whole = c.batch_of(np.concatenate([[0], np.cumsum(c.lens)]), sum(c.lens), max(c.lens))
    ko, vo = c.up(np.zeros((sum(c.lens), 3, dim), np.float32)), c.up(np.zeros((sum(c.lens), 3, dim), np.float32))
    eng.kv4_gather_dev(c.cache, whole, ko.ptr, vo.ptr, L.DT_F32)
    eng.sync()
    np.testing.assert_array_equal(ko.download(np.float32, (sum(c.lens), 3, dim)), np.concatenate([k_want[b] for b in total]))
    np.testing.assert_array_equal(vo.download(np.float32, (sum(c.lens), 3, dim)), np.concatenate([v_want[b] for b in total]))
    # the page format itself, decoded byte by byte
    raw = c.pages.download(np.uint8, (c.bytes,))
    for b, p, h in ((0, 69, 2), (0, 37, 0), (1, 4, 1), (2, 0, 2)):
        kk, vv = R.decode_position(raw, c.table, b, p, h, 3, dim, 16)
        np.testing.assert_array_equal(kk, k_want[b][p, h])
        np.testing.assert_array_equal(vv, v_want[b][p, h])
    c.free()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim,kv_heads,rotary,interleaved", [(64, 8, 32, 1), (64, 7, 64, 0), (128, 8, 0, 0), (256, 6, 64, 0), (256, 4, 256, 1)])
def test_append_many_rows(eng, dim, kv_heads, rotary, interleaved, dtype):
    """Enough rows for several heads to a CTA; first and last positions inside quads and pages."""
    c = Case(eng, [1813, 1502], [1810, 1502], kv_heads=kv_heads, dim=dim, page=48, seed=dim + kv_heads)
    k = as_type(c.rng.standard_normal((c.rows, kv_heads, dim)), dtype)
    v = as_type(c.rng.standard_normal((c.rows, kv_heads, dim)), dtype)
    pos = c.rng.integers(0, 4000, c.rows).astype(np.int32)
    tab = rope_table(rotary, 4000, 1e4, scaling=L.ROPE_NTK, factor=2.0) if rotary else None
    eng.kv4_append_dev(c.cache, c.batch, c.up(k).ptr, c.up(v).ptr, dtype, rope=RopeTable(c.up(tab).ptr, 4000, rotary, interleaved) if rotary else None,
                       rope_positions=c.up(pos).ptr if rotary else 0)
    ko, vo = c.up(np.zeros((c.rows, kv_heads, dim), np.float32)), c.up(np.zeros((c.rows, kv_heads, dim), np.float32))
    eng.kv4_gather_dev(c.cache, c.batch, ko.ptr, vo.ptr, L.DT_F32)
    eng.sync()
    kf, vf = as_f64(k, dtype).astype(np.float32), as_f64(v, dtype).astype(np.float32)
    np.testing.assert_array_equal(ko.download(np.float32, k.shape), R.codec(R.rotate_f32(kf, tab[pos], interleaved) if rotary else kf))
    np.testing.assert_array_equal(vo.download(np.float32, k.shape), R.codec(vf))
    c.free()


def test_append_leaves_other_positions(eng):
    c = Case(eng, [40, 21], [3, 2], kv_heads=2, dim=128, page=16, seed=5)
    c.fill()
    before = c.pages.download(np.uint8, (c.bytes,))
    kv = np.ones((5, 2, 128), np.float32)
    eng.kv4_append_dev(c.cache, c.batch, c.up(kv).ptr, c.up(kv).ptr, L.DT_F32)
    eng.sync()
    after = c.pages.download(np.uint8, (c.bytes,))
    owner = R.owners(c.table, c.lens, c.num_pages, 2, 128, 16)  # (sequence, position) of every byte, -1 outside
    first = np.array([n - q for n, q in zip(c.lens, c.q_lens)] + [1 << 30])
    touched = owner[:, 1] >= first[owner[:, 0]]
    assert np.array_equal(before[~touched], after[~touched])
    assert not np.array_equal(before[touched], after[touched])
    c.free()


def test_strides_alignment_and_positions(eng):
    """Keys and values as slices of one fused projection, at odd offsets, rotated by positions of the caller's own."""
    c = Case(eng, [30], [30], kv_heads=2, dim=64, page=16, seed=9)
    for dtype in (L.DT_F32, L.DT_BF16):
        for off, row in ((0, 300), (3, 301), (1, 517)):
            x = as_type(c.rng.standard_normal((30, row)), dtype)
            item = x.dtype.itemsize
            tab = rope_table(48, 600, 1e4, scaling=L.ROPE_LINEAR, factor=4.0)
            pos = c.rng.integers(0, 600, 30).astype(np.int32)
            buf = c.up(x)
            eng.kv4_append_dev(c.cache, c.batch, buf.ptr + off * item, buf.ptr + (off + 130) * item, dtype,
                               rope=RopeTable(c.up(tab).ptr, 600, 48, 0), rope_positions=c.up(pos).ptr, k_strides=(row, 64), v_strides=(row, 70))
            ko, vo = c.up(np.zeros((30, 2, 64), np.float32)), c.up(np.zeros((30, 2, 64), np.float32))
            eng.kv4_gather_dev(c.cache, c.batch, ko.ptr, vo.ptr, L.DT_F32)
            eng.sync()
            f = as_f64(x, dtype).astype(np.float32)
            kf = f[:, off:off + 128].reshape(30, 2, 64)
            vf = np.stack([f[:, off + 130:off + 194], f[:, off + 200:off + 264]], 1)
            np.testing.assert_array_equal(ko.download(np.float32, (30, 2, 64)), R.codec(R.rotate_f32(kf, tab[pos], 0)))
            np.testing.assert_array_equal(vo.download(np.float32, (30, 2, 64)), R.codec(vf))
    c.free()


def test_non_finite_values(eng):
    """A group that holds an infinity or NaN reads back as NaN, its neighbours as they are; a hidden position with such a
    group does not reach a result."""
    c = Case(eng, [8], [8], kv_heads=1, dim=128, page=16, seed=2)
    k = c.rng.standard_normal((8, 1, 128)).astype(np.float32)
    v = k.copy()
    for p, bad in ((1, np.nan), (3, np.inf), (5, -np.inf)):
        k[p, 0, 70] = bad
        v[p, 0, 3] = bad
    eng.kv4_append_dev(c.cache, c.batch, c.up(k).ptr, c.up(v).ptr, L.DT_F32)
    ko, vo = c.up(np.zeros((8, 1, 128), np.float32)), c.up(np.zeros((8, 1, 128), np.float32))
    eng.kv4_gather_dev(c.cache, c.batch, ko.ptr, vo.ptr, L.DT_F32)
    q = c.rng.standard_normal((8, 1, 128)).astype(np.float32)
    out = c.up(np.zeros_like(q))
    eng.kv4_attention_dev(c.cache, c.batch, c.up(q).ptr, out.ptr, L.DT_F32, 1, scale=0.1)
    eng.sync()
    kg, vg = ko.download(np.float32, k.shape), vo.download(np.float32, v.shape)
    bad = [1, 3, 5]
    good = [0, 2, 4, 6, 7]
    assert np.isnan(kg[bad, 0, 64:]).all() and np.isnan(vg[bad, 0, :64]).all()
    np.testing.assert_array_equal(kg[good], R.codec(k[good]))
    np.testing.assert_array_equal(kg[:, 0, :64], R.codec(np.ascontiguousarray(k[:, 0, :64])))
    got = out.download(np.float32, q.shape)
    assert np.isfinite(got[0]).all() and np.isnan(got[1:]).all()
    c.free()


def test_non_finite_values_in_a_prompt(eng):
    """The same for many bf16 rows: rows before the position (or with it outside their window) keep their results."""
    c = Case(eng, [300], [300], kv_heads=1, dim=128, page=16, seed=2)
    k = c.rng.standard_normal((300, 1, 128)).astype(np.float32)
    v = c.rng.standard_normal((300, 1, 128)).astype(np.float32)
    v[170, 0, 5] = np.inf
    eng.kv4_append_dev(c.cache, c.batch, c.up(k).ptr, c.up(v).ptr, L.DT_F32)
    q = as_type(c.rng.standard_normal((300, 4, 128)), L.DT_BF16)
    out = c.up(np.zeros_like(q))
    v[170] = 0.0
    for window in (0, 20):
        eng.kv4_attention_dev(c.cache, c.batch, c.up(q).ptr, out.ptr, L.DT_BF16, 4, scale=0.1, window=window)
        eng.sync()
        got = as_f64(out.download(q.dtype, q.shape), L.DT_BF16)
        hit = np.arange(300) >= 170 if window == 0 else (np.arange(300) >= 170) & (np.arange(300) < 190)
        assert np.isnan(got[hit][..., :64]).all() and np.isfinite(got[~hit]).all()
        want, size, reach = R.attention(as_f64(q, L.DT_BF16), R.codec(k), R.codec(v), [300], [300], window, 0.1)
        assert np.all(np.abs(got - want)[~hit] <= bound_of(L.DT_BF16, want, size, reach)[~hit])
    c.free()


# ─── rotary positions ───────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("dim,rotary,heads,gap,off", [(256, 64, 16, 256, 0), (128, 128, 3, 0, 0), (64, 16, 1, 0, 0), (96, 42, 5, 7, 1), (64, 2, 2, 0, 3),
                                                      (33, 30, 2, 1, 0)])
def test_rope(eng, dim, rotary, heads, gap, off, interleaved, dtype):
    rng = np.random.default_rng(dim + rotary)
    for n in (1, 9, 700):
        stride = dim + gap
        x = as_type(rng.standard_normal(off + n * heads * stride), dtype)
        pos = rng.integers(0, 5000, n).astype(np.int32)
        tab = rope_table(rotary, 5000, 1e7, scaling=L.ROPE_YARN, factor=4.0, original_positions=1024)
        xb, pb, tb = (eng.alloc(a.nbytes).upload(a) for a in (x, pos, tab))
        ob = eng.alloc(n * heads * dim * x.dtype.itemsize)
        rope = RopeTable(tb.ptr, 5000, rotary, interleaved)
        eng.rope_dev(rope, xb.ptr + off * x.dtype.itemsize, ob.ptr, pb.ptr, dtype, n, heads, dim, x_strides=(heads * stride, stride))
        eng.sync()
        src = as_f64(x[off:].reshape(n, heads, stride)[..., :dim], dtype).astype(np.float32)
        want = as_type(R.rotate_f32(src, tab[pos], interleaved), dtype)
        np.testing.assert_array_equal(ob.download(x.dtype, (n, heads, dim)), want)
        # in place
        eng.rope_dev(rope, xb.ptr + off * x.dtype.itemsize, xb.ptr + off * x.dtype.itemsize, pb.ptr, dtype, n, heads, dim,
                     x_strides=(heads * stride, stride), out_strides=(heads * stride, stride))
        eng.sync()
        after = xb.download(x.dtype, x.shape)[off:].reshape(n, heads, stride)
        np.testing.assert_array_equal(after[..., :dim], want)
        np.testing.assert_array_equal(after[..., dim:], x[off:].reshape(n, heads, stride)[..., dim:])
        for buf in (xb, pb, tb, ob):
            buf.free()


# ─── all of them, as a decode loop uses them ────────────────────────────────
def test_prompt_then_decode(eng):
    """Two sequences: a prompt each, then five decode steps; queries rotated, keys rotated on the way into the cache."""
    heads, kv_heads, dim, rotary, page = 4, 2, 128, 64, 16
    c = Case(eng, [60, 43], [55, 38], kv_heads=kv_heads, dim=dim, page=page, seed=21)
    tab = rope_table(rotary, 64, 1e4)
    rope = RopeTable(c.up(tab).ptr, 64, rotary, 0)
    q_all, k_all, v_all = (c.rng.standard_normal((2, 60, h, dim)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    for step in range(6):
        lens = [55 + step, 38 + step]
        q_lens = [55, 38] if step == 0 else [1, 1]
        take = lambda x: np.concatenate([x[b, lens[b] - q_lens[b]:lens[b]] for b in range(2)])  # noqa: E731
        q, k, v = take(q_all), take(k_all), take(v_all)
        pos = np.concatenate([np.arange(lens[b] - q_lens[b], lens[b]) for b in range(2)]).astype(np.int32)
        batch = c.batch_of(np.concatenate([[0], np.cumsum(q_lens)]), sum(q_lens), max(q_lens), lens)
        qb, out = c.up(q), c.up(np.zeros_like(q))
        eng.rope_dev(rope, qb.ptr, qb.ptr, c.up(pos).ptr, L.DT_F32, sum(q_lens), heads, dim)
        eng.kv4_append_dev(c.cache, batch, c.up(k).ptr, c.up(v).ptr, L.DT_F32, rope=rope)
        eng.kv4_attention_dev(c.cache, batch, qb.ptr, out.ptr, L.DT_F32, heads, scale=1 / math.sqrt(dim))
        eng.sync()
        kk = np.concatenate([R.codec(R.rotate_f32(k_all[b, :lens[b]], tab[:lens[b]], 0)) for b in range(2)])
        vv = np.concatenate([R.codec(np.ascontiguousarray(v_all[b, :lens[b]])) for b in range(2)])
        want, size, reach = R.attention(R.rotate_f32(q, tab[pos], 0).astype(np.float64), kk, vv, lens, q_lens, 0, 1 / math.sqrt(dim))
        assert np.all(np.abs(out.download(np.float32, q.shape) - want) <= bound_of(L.DT_F32, want, size, reach))
    c.free()


# ─── what the device reports ────────────────────────────────────────────────
def test_bad_entries_are_reported_and_touch_nothing(eng):
    c = Case(eng, [40, 20], [2, 1], kv_heads=2, dim=64, page=16, seed=4)
    c.fill()
    before = c.pages.download(np.uint8, (c.bytes,))
    kv = c.up(np.ones((3, 2, 64), np.float32))
    q, out, out2 = c.up(np.ones((3, 2, 64), np.float32)), c.up(np.zeros((3, 2, 64), np.float32)), c.up(np.zeros((3, 2, 64), np.float32))
    tab = RopeTable(c.up(rope_table(8, 30, 1e4)).ptr, 30, 8, 0)
    for bad in (-5, c.num_pages, 1 << 30):
        saved = c.table.copy()
        c.table[0, 2], c.table[1, 1] = bad, bad
        batch = c.batch_of(c.q_start, 3, 2)
        c.table = saved
        for call in (lambda: eng.kv4_append_dev(c.cache, batch, kv.ptr, kv.ptr, L.DT_F32),
                     lambda: eng.kv4_gather_dev(c.cache, batch, out.ptr, out2.ptr, L.DT_F32),
                     lambda: eng.kv4_attention_dev(c.cache, batch, q.ptr, out.ptr, L.DT_F32, 2, scale=0.1)):
            call()
            with pytest.raises(ValueError, match="page table"):
                eng.sync()
    for q_start, lens in (([0, 2, 9], [40, 20]), ([0, 3, 2], [40, 20]), ([0, 2, 3], [40, 900]), ([0, 2, 3], [-1, 20])):
        batch = c.batch_of(q_start, 3, 2, lens)
        batch.max_seq_len = 40
        if lens[0] == 40 and lens[1] == 20:
            eng.kv4_append_dev(c.cache, batch, kv.ptr, kv.ptr, L.DT_F32)
            with pytest.raises(ValueError, match="q_start or seq_lens"):
                eng.sync()
            c.pages.upload(before)
        eng.kv4_attention_dev(c.cache, batch, q.ptr, out.ptr, L.DT_F32, 2, scale=0.1)
        with pytest.raises(ValueError, match="q_start or seq_lens"):
            eng.sync()
    eng.rope_dev(tab, q.ptr, out.ptr, c.up(np.array([0, 30, -1], np.int32)).ptr, L.DT_F32, 3, 2, 64)
    with pytest.raises(ValueError, match="rotary table"):
        eng.sync()
    assert np.array_equal(before, c.pages.download(np.uint8, (c.bytes,)))
    eng.kv4_attention_dev(c.cache, c.batch, q.ptr, out.ptr, L.DT_F32, 2, scale=0.1)
    eng.sync()  # and the engine carries on
    c.free()
