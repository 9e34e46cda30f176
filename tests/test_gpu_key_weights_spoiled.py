"""What a NaN or an infinity in a query or in a key's scale does to the weight that cached keys
receive: all weights of its sequence and KV head become NaN, whichever form of the kernels the
batch's rows and bounds choose, and no others change by a bit."""
import numpy as np
import pytest

import paged_oracle as po
from test_gpu_key_weights import run
from test_gpu_paged_q8 import Batch

pytestmark = pytest.mark.gpu

SPOILS = [np.nan, np.inf, -np.inf]
# (new tokens, tokens before, query heads of a KV head, window, bound of keys or none).
FORMS = {
    "single tokens": ([1, 1, 2], [300, 33, 700], 2, 0, None),
    "up to sixteen rows": ([3, 2, 1], [300, 33, 700], 5, 0, None),
    "few rows beside many": ([1, 40, 2], [300, 90, 700], 4, 0, 1 << 19),
    "chunks": ([70, 40, 130], [30, 0, 500], 2, 0, None),
    "one chunk": ([300], [40], 2, 0, None),
    "windows": ([70, 40, 130], [30, 0, 500], 2, 37, None),
    "many tokens": ([1] * 40 + [30], [64] * 40 + [9], 2, 0, None),
}


def scene(form, f16, signed):
    """`signed`: queries above zero and keys below, so that each product is negative: an
    infinite factor makes it -inf."""
    new, before, group, window, bound = FORMS[form]
    rng = np.random.default_rng(40 + len(form))
    batch = Batch(rng, 16, new, before, gap=2)
    kv, d = 2, 64
    cache = po.Pages(rng, batch.pages, 16, kv, d)
    query = rng.standard_normal((batch.tokens, group * kv, d))
    if signed:
        query = np.abs(query)
        cache.codes["key"][:] = -np.abs(cache.codes["key"].astype(int)).clip(1, 127)
    stride = int(batch.lengths.max()) + 3
    if bound:
        table = np.full((len(new), bound // 16), -1, np.int32)
        table[:, :batch.width] = batch.table
        batch.table, batch.width, batch.max_keys, stride = table, bound // 16, 1 << 30, bound
        # (Keys of 64 MB by the bounds: launches of their own for sequences of few rows.)
        assert len(new) * kv * bound * d > 64e6
    old = np.zeros((len(new), kv, stride), np.float32)
    old[..., :900] = rng.random(old[..., :900].shape)
    return batch, cache, query.astype(np.float16 if f16 else np.float32), old, group, window


def check(got, want, batch, spoiled):
    """spoiled: pairs (sequence, KV head)."""
    for b, length in enumerate(batch.lengths):
        for h in range(got.shape[1]):
            if (b, h) in spoiled:
                assert np.isnan(got[b, h, :length]).all(), (
                    b, h, int((~np.isnan(got[b, h, :length])).sum()), int(length))
                np.testing.assert_array_equal(got[b, h, length:], want[b, h, length:])
            else:
                np.testing.assert_array_equal(got[b, h], want[b, h])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_of_a_query(hip_ctx, form, f16):
    """In the first row that counts, which sees the fewest keys, and in the last."""
    for signed in (False, True):
        batch, cache, query, old, group, window = scene(form, f16, signed)
        want = run(hip_ctx, cache, batch, 2 * group, query, old, window, 0.5)
        assert np.isfinite(want).all()
        for b in (0, len(batch.new) - 1):
            n = int(batch.new[b])
            for row in (n - min(n, window or n), n - 1):
                for value in SPOILS:
                    bad = query.copy()
                    bad[int(batch.starts[b]) + row, 2 * group - 1, 5] = value
                    got = run(hip_ctx, cache, batch, 2 * group, bad, old, window, 0.5)
                    check(got, want, batch, {(b, 1)})


@pytest.mark.parametrize("f16", [False, True])
def test_of_a_query_before_the_window(hip_ctx, f16):
    """Rows that do not count spoil nothing."""
    batch, cache, query, old, group, window = scene("windows", f16, True)
    want = run(hip_ctx, cache, batch, 2 * group, query, old, window, 0.5)
    bad = query.copy()
    for b, n in enumerate(batch.new):
        bad[int(batch.starts[b]):int(batch.starts[b]) + n - min(n, window)] = np.inf
    got = run(hip_ctx, cache, batch, 2 * group, bad, old, window, 0.5)
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_of_a_scale(hip_ctx, form, f16):
    """Of the first page and of the last, which the first rows may not see."""
    for signed in (False, True):
        batch, cache, query, old, group, window = scene(form, f16, signed)
        want = run(hip_ctx, cache, batch, 2 * group, query, old, window, 0.0)
        for b in (0, len(batch.new) - 1):
            last = -(-int(batch.lengths[b]) // 16) - 1
            for page in (batch.table[b, 0], batch.table[b, last]):
                held = cache.scales["key"][page, 0]
                for value in (np.nan, np.inf):
                    cache.scales["key"][page, 0] = value
                    got = run(hip_ctx, cache, batch, 2 * group, query, old, window, 0.0)
                    check(got, want, batch, {(b, 0)})
                cache.scales["key"][page, 0] = held


@pytest.mark.parametrize("f16", [False, True])
def test_across_groups_of_rows(hip_ctx, f16):
    """Bounds of a million keys: statistics of rows in groups (127 tokens here); a row of the
    first group spoils what later ones add to."""
    rng = np.random.default_rng(47)
    batch = Batch(rng, 64, [200, 1, 70], [100, 300, 90], gap=3)
    cache = po.Pages(rng, batch.pages, 64, 1, 64)
    stride = 1 << 20
    table = np.full((3, stride // 64), -1, np.int32)
    table[:, :batch.width] = batch.table
    batch.table, batch.width, batch.max_keys = table, stride // 64, 1 << 30
    query = rng.standard_normal((batch.tokens, 64, 64)).astype(np.float16 if f16 else np.float32)
    old = np.zeros((3, 1, stride), np.float32)
    old[..., :400] = rng.random((3, 1, 400))
    want = run(hip_ctx, cache, batch, 64, query, old, 0, 0.8)
    for value, b, row in ((np.nan, 0, 0), (np.inf, 0, 199), (-np.inf, 2, 0)):
        bad = query.copy()
        bad[int(batch.starts[b]) + row, 9, 3] = value
        got = run(hip_ctx, cache, batch, 64, bad, old, 0, 0.8)
        check(got, want, batch, {(b, 0)})
