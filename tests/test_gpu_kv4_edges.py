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
