"""The paged 8-bit KV cache at the ends of the numbers' ranges: pages of zeros beside
ordinary and very large ones, and rows at the least scale that a page holds.  The
tolerances are those of tests/test_gpu_paged_q8.py where no other is given.
"""
import math

import numpy as np
import pytest

import paged_oracle as po
from test_gpu_paged_q8 import Batch, DevicePages, run_attention, run_prologue

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -70  # the least scale of a page that is not all zeros


def pages_of_scores(rng, octaves, value_scales, head_dim=64, page_tokens=64):
    """A cache whose page i gives every key the score octaves[i] (in powers of two of the
    weight) for the query that is returned, and the values their scale."""
    n = len(octaves)
    cache = po.Pages(rng, n, page_tokens, 1, head_dim)
    cache.codes["key"][:] = 64
    cache.scales["key"][:, 0] = octaves
    cache.scales["value"][:, 0] = value_scales
    cache.codes["value"][np.asarray(value_scales) == 0] = 0
    return cache, math.sqrt(head_dim) * math.log(2) / (head_dim * 64.0)


def run_of_pages(cache, table, new):
    """A batch of one sequence over table's pages whose last `new` tokens are rows; its
    bounds so loose that the keys are not split further than they must be."""
    before = len(table) * cache.page_tokens - new
    batch = Batch(np.random.default_rng(0), cache.page_tokens, [new], [before])
    batch.table = np.array([table], np.int32)
    batch.max_query, batch.max_keys = 2 ** 31 - 1, 2 ** 31 - 1
    return batch


def check(ctx, cache, batch, level, kind):
    query = np.full((batch.tokens, 1, cache.head_dim), level, kind)
    got = run_attention(ctx, cache, batch, 1, query, f16=kind == np.float16)
    want, size, score = po.attention(cache, query, batch.plain(), 1)
    tol = po.attention_tolerance(size, want, score, cache.head_dim, kind == np.float16)
    off = np.abs(got - want) / tol
    assert (off <= 1).all(), (float(np.nanmax(off)), got[-1, 0, :3], want[-1, 0, :3])
    return want


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_long_run_of_zero_pages(hip_ctx, kind):
    """33 rows over 20480 keys of zero values, whose scores lie just under four octaves
    above those of the first keys, and then ordinary values with about half the weight:
    the softmax's sum holds all of them."""
    rng = np.random.default_rng(60)
    cache, level = pages_of_scores(rng, [10.0, 13.9, 23.9], [0.0, 0.0, 0.03])
    batch = run_of_pages(cache, [0] + [1] * 320 + [2], 33)
    check(hip_ctx, cache, batch, level, kind)


@pytest.mark.parametrize("new", [1, 33])
def test_zero_pages_beside_large_values(hip_ctx, new):
    """32768 keys of zero values 17.5 octaves below a page of values near 2^30: together
    they have up to a seventh of the weight."""
    rng = np.random.default_rng(61)
    cache, level = pages_of_scores(rng, [5.0, 22.5], [0.0, 2.0 ** 24])
    batch = run_of_pages(cache, [0] * 512 + [1], new)
    check(hip_ctx, cache, batch, level, np.float32)


def test_rows_at_the_least_scale(hip_ctx):
    """Rows that need less than the least scale are held as zeros, those just above it as
    they are; one page each."""
    rng = np.random.default_rng(62)
    d, kv, pt = 64, 2, 16
    batch = Batch(rng, pt, [pt, pt, pt], [0, 0, 0])
    cache = po.Pages(rng, batch.pages, pt, kv, d)
    value = rng.uniform(-1, 1, (batch.tokens, kv, d)).astype(np.float32)
    value[:, :, 0] = 1.0  # the largest magnitude of every page and head
    sizes = [127.0 * LEAST * 0.99, 127.0 * LEAST * 1.01, 127.0 * LEAST * 2.0 ** -25]
    for b, size in enumerate(sizes):
        value[batch.starts[b]:batch.starts[b + 1]] *= np.float32(size)
    rows = {"q_gate": rng.standard_normal((batch.tokens, kv, 2, d)).astype(np.float32),
            "key": rng.standard_normal((batch.tokens, kv, d)).astype(np.float32), "value": value}
    pages = run_prologue(hip_ctx, rng, cache, batch, kv, 64, (11, 11, 10, 0), rows=rows)[4]
    got = pages.read()
    for b, kept in enumerate((False, True, False)):
        page = batch.table[b, 0]
        if kept:
            step = np.float32(value[batch.starts[b], 0, 0]) / np.float32(127)
            np.testing.assert_array_equal(got.scales["value"][page], step)
            assert (got.codes["value"][page, :, :, 0] == 127).all()
        else:
            assert (got.scales["value"][page] == 0).all()
            assert (got.codes["value"][page] == 0).all()


@pytest.mark.parametrize("size", [-1e6, 1e6])
@pytest.mark.parametrize("new,before", [([1], [0]), ([1, 1, 1], [5, 300, 0]), ([33], [0]),
                                        ([40, 1, 50], [70, 200, 0])])
def test_scores_at_the_end_of_their_range(hip_ctx, new, before, size):
    """Every key the same, with a score near size: a row's output is the mean of the
    values that it sees (to the f32 roundings of up to 300 equal weights, their codes' two
    f16 parts and the page scales' exponents beside a maximum of 2^20: its step is 1/8, but
    the same for all of them, 2^-17)."""
    rng = np.random.default_rng(63)
    d, pt = 64, 16
    batch = Batch(rng, pt, new, before)
    cache = po.Pages(rng, batch.pages, pt, 1, d)
    cache.codes["key"][:] = 100
    cache.scales["key"][:] = 3.0
    cache.scales["value"][:] = 0.03
    level = size / (d * 100.0 * 3.0) * math.sqrt(d)
    query = np.full((batch.tokens, 1, d), level, np.float32)
    got = run_attention(hip_ctx, cache, batch, 1, query)
    for b, count in enumerate(new):
        v = np.concatenate([cache.values_of("value", p) for p in batch.table[b] if p >= 0])[:, 0]
        for i in range(count):
            seen = v[:before[b] + i + 1]
            off = np.abs(got[int(batch.starts[b]) + i, 0] - seen.mean(0))
            assert (off <= 2.0 ** -17 * np.abs(seen).mean(0)).all(), (b, i)
