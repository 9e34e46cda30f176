"""The weight that cached keys receive, on the GPU against the plain 64-bit form
(tests/serving_oracle.py, which derives the tolerances)."""
import math

import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_gpu_paged_q8 import ATTEND_MIXES, HEADS, Batch, DevicePages

pytestmark = pytest.mark.gpu


def run(ctx, cache, batch, heads, query, old, window, decay):
    pages, tables = DevicePages(ctx, cache), batch.device(ctx)
    weights = ctx.buffer(old)
    call = (ctx.key_weights_f16q_paged_q8_kv if query.dtype == np.float16
            else ctx.key_weights_f32_paged_q8_kv)
    call(ctx.buffer(query), pages.struct, tables, heads, window, decay, weights, old.shape[2])
    return weights.download().reshape(old.shape)


def check(ctx, rng, cache, batch, heads, f16, window=0, decay=0.9, stride=None, spread=2.0,
          query=None):
    stride = stride or int(batch.lengths.max()) + 3
    if query is None:
        query = spread * rng.standard_normal((batch.tokens, heads, cache.head_dim))
    query = query.astype(np.float16 if f16 else np.float32)
    old = rng.random((len(batch.new), cache.kv_heads, stride)).astype(np.float32)
    got = run(ctx, cache, batch, heads, query, old, window, decay)
    want, tol = so.key_weights(cache, query, batch.plain(), heads, window, decay, old, stride)
    untouched = tol == 0
    np.testing.assert_array_equal(got[untouched], old[untouched])
    off = np.abs(got - want)[~untouched] / tol[~untouched]
    assert (off <= 1).all(), (off.max(), np.argwhere(~(np.abs(got - want) <= tol))[:4])
    return got


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mix", ATTEND_MIXES)
@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("d,heads,kv_heads", HEADS)
def test_matches_plain(hip_ctx, d, heads, kv_heads, page_tokens, mix, f16):
    rng = np.random.default_rng(d + heads + page_tokens)
    batch = Batch(rng, page_tokens, *ATTEND_MIXES[mix], gap=1)
    cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
    check(hip_ctx, rng, cache, batch, heads, f16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window", [1, 3, 32, 33, 64, 1000])
def test_windows(hip_ctx, window, f16):
    rng = np.random.default_rng(window)
    batch = Batch(rng, 32, [150, 1, 31, 0, 64], [700, 90, 0, 12, 129])
    cache = po.Pages(rng, batch.pages, 32, 2, 128)
    check(hip_ctx, rng, cache, batch, 8, f16, window=window, decay=1.0)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,heads,kv_heads,page_tokens", [(256, 16, 1, 32), (128, 5, 5, 128),
                                                         (64, 24, 2, 128), (128, 34, 2, 32)])
def test_group_sizes(hip_ctx, d, heads, kv_heads, page_tokens, f16):
    rng = np.random.default_rng(d + heads)
    for new, before in (([1, 1], [400, 3]), ([9, 1, 70], [0, 333, 129])):
        batch = Batch(rng, page_tokens, new, before)
        cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
        check(hip_ctx, rng, cache, batch, heads, f16)


@pytest.mark.parametrize("new,before,f16", [([1], [40000], False), ([1, 1], [33000, 9], True),
                                            ([300], [5000], False), ([700], [0], True),
                                            ([40, 500], [9000, 100], False)])
def test_long_contexts(hip_ctx, new, before, f16):
    rng = np.random.default_rng(before[0])
    batch = Batch(rng, 64, new, before)
    cache = po.Pages(rng, batch.pages, 64, 1, 128)
    check(hip_ctx, rng, cache, batch, 4, f16, window=0 if sum(new) < 10 else 37)


def test_weights_sum_to_the_rows(hip_ctx):
    """With decay 0 the keys of a KV head receive one unit from each row, whatever the
    memory held."""
    rng = np.random.default_rng(5)
    batch = Batch(rng, 64, [1, 17, 300], [900, 0, 4000])
    cache = po.Pages(rng, batch.pages, 64, 2, 256)
    old = np.full((3, 2, 4300), np.nan, np.float32)
    query = (2 * rng.standard_normal((batch.tokens, 8, 256))).astype(np.float32)
    got = run(hip_ctx, cache, batch, 8, query, old, 0, 0.0)
    for b, (n, length) in enumerate(zip(batch.new, batch.lengths)):
        np.testing.assert_allclose(got[b, :, :length].astype(np.float64).sum(-1), 4 * n, rtol=1e-5)
        assert np.isnan(got[b, :, length:]).all()


def test_new_positions_have_no_earlier_weight(hip_ctx):
    """What lies behind the tokens before is not read, a NaN not either."""
    rng = np.random.default_rng(6)
    for new, before in (([3], [40]), ([60], [100])):
        batch = Batch(rng, 16, new, before)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        old = rng.random((1, 2, 200)).astype(np.float32)
        old[..., before[0]:] = np.nan
        query = rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)
        got = run(hip_ctx, cache, batch, 4, query, old, 0, 1.0)
        clean = np.where(np.isnan(old), 0, old)
        want, tol = so.key_weights(cache, query, batch.plain(), 4, 0, 1.0, clean, 200)
        n = int(batch.lengths[0])
        assert (np.abs(got - want)[..., :n] <= tol[..., :n]).all()
        assert np.isnan(got[..., n:]).all()


@pytest.mark.parametrize("spoil", ["length", "query", "width", "stride", "starts"])
def test_leaves_out_what_breaks_a_bound(hip_ctx, spoil):
    rng = np.random.default_rng(12)
    batch = Batch(rng, 16, [3, 20, 4], [10, 30, 13], gap=1)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    stride = 60
    if spoil == "length":
        batch.max_keys = 40
    elif spoil == "query":
        batch.max_query = 8
    elif spoil == "width":
        batch.lengths[1] = 16 * batch.width + 1
        batch.max_keys, stride = 1000, 1000
    elif spoil == "stride":
        stride = 45
    else:
        batch.starts[2] = 1
    check(hip_ctx, rng, cache, batch, 4, False, stride=stride)


@pytest.mark.parametrize("f16", [False, True])
def test_pages_outside_the_pool(hip_ctx, f16):
    """Their keys receive nothing; a row that sees no others gives nothing."""
    rng = np.random.default_rng(13)
    batch = Batch(rng, 16, [1, 40, 2, 5], [100, 200, 3, 8])
    cache = po.Pages(rng, batch.pages, 16, 2, 128)
    batch.table[0, [1, 3]] = [-1, cache.pages]
    batch.table[1, :11] = 2 ** 31 - 1
    batch.table[2, 0] = -7
    got = check(hip_ctx, rng, cache, batch, 4, f16, decay=0.0)
    assert (got[2, :, :5] == 0).all() and (got[0, :, 16:32] == 0).all()


@pytest.mark.parametrize("f16", [False, True])
def test_queries_and_scales_out_of_the_ordinary(hip_ctx, f16):
    """Zero and huge queries, zero and far apart scales; a NaN stays with its KV head."""
    rng = np.random.default_rng(14)
    for new, before in (([1, 1, 1], [90, 300, 33]), ([70, 40, 1], [30, 0, 500])):
        batch = Batch(rng, 16, new, before)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        cache.scales["key"][:] = rng.choice([0.0, 1e-30, 1e-6, 0.03, 1.0], cache.scales["key"].shape)
        query = rng.standard_normal((batch.tokens, 4, 64)) * rng.choice(
            [0.0, 1e-4, 1.0, 30.0], (batch.tokens, 4, 1))
        check(hip_ctx, rng, cache, batch, 4, f16, query=query)
        kind = np.float16 if f16 else np.float32
        clean = rng.standard_normal((batch.tokens, 4, 64)).astype(kind)
        old = rng.random((3, 2, 600)).astype(np.float32)
        want = run(hip_ctx, cache, batch, 4, clean, old, 0, 0.5)
        spoiled = clean.copy()
        spoiled[batch.starts[1], 3, 5] = np.nan
        cache.scales["key"][batch.table[0, 1], 0] = np.nan
        got = run(hip_ctx, cache, batch, 4, spoiled, old, 0, 0.5)
        n = batch.lengths
        visible = int(before[1]) + 1
        assert np.isnan(got[0, 0, :n[0]]).all() and np.isnan(got[1, 1, :visible]).all()
        for b, h in ((0, 1), (1, 0), (2, 0), (2, 1)):
            np.testing.assert_array_equal(got[b, h], want[b, h])


def test_pages_may_be_shared_and_bounds_loose(hip_ctx):
    rng = np.random.default_rng(15)
    batch = Batch(rng, 16, [1, 60, 3], [200, 150, 180])
    batch.table[1, :8] = batch.table[0, :8]
    batch.table[2, :8] = batch.table[0, :8]
    batch.max_query = batch.max_keys = 2 ** 31 - 1
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    check(hip_ctx, rng, cache, batch, 6, False)
    check(hip_ctx, rng, cache, batch, 6, True, window=2)


@pytest.mark.parametrize("sequences", [65, 130])
def test_many_sequences(hip_ctx, sequences):
    rng = np.random.default_rng(sequences)
    new = rng.integers(0, 30, sequences)
    new[::3] = 1
    batch = Batch(rng, 16, new.tolist(), rng.integers(0, 500, sequences).tolist(), gap=2)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    check(hip_ctx, rng, cache, batch, 6, sequences % 2 == 0, window=20)


def test_the_same_bits_in_any_batch(hip_ctx):
    """A sequence's weights do not depend on what else the batch holds."""
    rng = np.random.default_rng(16)
    new, before = [1, 40, 1], [500, 300, 20]
    batch = Batch(rng, 16, new, before)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    query = rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)
    old = rng.random((3, 2, 600)).astype(np.float32)
    first = run(hip_ctx, cache, batch, 4, query, old, 0, 0.5)
    np.testing.assert_array_equal(first, run(hip_ctx, cache, batch, 4, query, old, 0, 0.5))


@pytest.mark.parametrize("max_query", [1, 80])
def test_captured_call_replays(hip_ctx, max_query):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(17)
    d, heads, kv, pt, tokens = 128, 8, 2, 16, 90
    cache = po.Pages(rng, 130, pt, kv, d)
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    t = {"keys": torch.from_numpy(cache.codes["key"]).cuda(),
         "values": torch.from_numpy(cache.device_values()).cuda(),
         "ks": torch.from_numpy(cache.scales["key"]).cuda(),
         "vs": torch.from_numpy(cache.scales["value"]).cuda(),
         "table": torch.zeros(3, 40, dtype=torch.int32, device="cuda"),
         "starts": torch.zeros(4, dtype=torch.int32, device="cuda"),
         "lengths": torch.zeros(3, dtype=torch.int32, device="cuda"),
         "q": torch.zeros(tokens, heads, d, device="cuda"),
         "w": torch.zeros(3, kv, 640, device="cuda"),
         "w2": torch.zeros(3, kv, 640, device="cuda")}
    b = {n: kh.as_buffer(x) for n, x in t.items()}
    pages = kh.PagedQ8Cache(b["keys"], b["values"], b["ks"], b["vs"], 130, pt, kv, d)
    batch = kh.PagedBatch(b["table"], b["starts"], b["lengths"], 3, 40, tokens, max_query, 640)

    def call(out):
        ctx.key_weights_f32_paged_q8_kv(b["q"], pages, batch, heads, 0, 0.5, b[out], 640)

    sets = [([1, 1, 1], [600, 30, 0]), ([1, 0, 1], [5, 100, 639]), ([1, 1, 1], [63, 64, 65])]
    if max_query > 1:
        sets += [([80, 1, 4], [500, 7, 100]), ([2, 70, 1], [0, 570, 300])]
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call("w")
        for new, before in sets:
            lengths = [x + y for x, y in zip(new, before)]
            t["table"].copy_(torch.from_numpy(rng.permutation(130)[:120].reshape(3, 40)))
            t["starts"].copy_(torch.tensor([0, *np.cumsum(new)]))
            t["lengths"].copy_(torch.tensor(lengths))
            t["q"].copy_(torch.from_numpy(rng.standard_normal((tokens, heads, d))))
            old = torch.rand(3, kv, 640, device="cuda")
            t["w"].copy_(old)
            t["w2"].copy_(old)
            graph.replay()
            call("w2")
            stream.synchronize()
            assert torch.equal(t["w"], t["w2"])
            assert not torch.equal(t["w"], old)
    ctx.commit_graph()
    ctx.close()


def test_two_steps_add_up(hip_ctx):
    """Two decode steps with decay 1 receive what the two-token batch does."""
    rng = np.random.default_rng(18)
    cache = po.Pages(rng, 9, 64, 2, 64)
    table = rng.permutation(9)[:5].reshape(1, 5).astype(np.int32)
    query = rng.standard_normal((2, 4, 64)).astype(np.float32)
    batch = Batch(rng, 64, [2], [200])
    batch.table, batch.width, batch.pages = table, 5, 9
    start = np.zeros((1, 2, 300), np.float32)
    both = run(hip_ctx, cache, batch, 4, query, start, 0, 1.0)
    have = start
    for i in range(2):
        one = Batch(rng, 64, [1], [200 + i])
        one.table, one.width, one.pages = table, 5, 9
        have = run(hip_ctx, cache, one, 4, query[i:i + 1], have, 0, 1.0)
    np.testing.assert_allclose(have, both, rtol=2e-6, atol=1e-12)
    assert math.isclose(float(both.sum()), 2 * 4, rel_tol=1e-5)


@pytest.mark.parametrize("window", [0, 150])
def test_groups_of_rows(hip_ctx, window):
    """Bounds of a million keys: statistics of rows in groups (127 tokens here), which a
    sequence's rows lie across, its earlier weight decayed once."""
    rng = np.random.default_rng(19)
    batch = Batch(rng, 64, [200, 1, 30, 0, 70], [100, 300, 0, 40, 90], gap=3)
    cache = po.Pages(rng, batch.pages, 64, 1, 64)
    stride = 1 << 20
    table = np.full((5, stride // 64), -1, np.int32)
    table[:, :batch.width] = batch.table
    batch.table, batch.width, batch.max_keys = table, stride // 64, 1 << 30
    query = rng.standard_normal((batch.tokens, 64, 64)).astype(np.float32)
    old = np.zeros((5, 1, stride), np.float32)
    old[..., :400] = rng.random((5, 1, 400))
    got = run(hip_ctx, cache, batch, 64, query, old, window, 0.8)
    want, tol = so.key_weights(cache, query, batch.plain(), 64, window, 0.8, old, stride)
    untouched = tol == 0
    assert np.array_equal(got[untouched], old[untouched])
    off = np.abs(got - want)[~untouched] / tol[~untouched]
    assert (off <= 1).all(), off.max()


def test_bounds_too_loose_to_keep_scores(hip_ctx):
    """Single tokens whose scores would take more than 1 GiB, as far as the bounds say."""
    rng = np.random.default_rng(20)
    batch = Batch(rng, 64, [1, 1, 2, 1], [100, 300, 7, 0])
    cache = po.Pages(rng, batch.pages, 64, 4, 64)
    stride = 1 << 21
    table = np.full((4, stride // 64), -1, np.int32)
    table[:, :batch.width] = batch.table
    batch.table, batch.width, batch.max_keys = table, stride // 64, 1 << 30
    query = rng.standard_normal((batch.tokens, 64, 64)).astype(np.float32)
    old = np.zeros((4, 4, stride), np.float32)
    old[..., :400] = rng.random((4, 4, 400))
    got = run(hip_ctx, cache, batch, 64, query, old, 0, 0.8)
    want, tol = so.key_weights(cache, query, batch.plain(), 64, 0, 0.8, old, stride)
    untouched = tol == 0
    assert np.array_equal(got[untouched], old[untouched])
    off = np.abs(got - want)[~untouched] / tol[~untouched]
    assert (off <= 1).all(), off.max()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 256])
def test_few_and_many_rows_in_one_call(hip_ctx, d, f16):
    """Bounds of so many keys that sequences of few rows have their own launches beside
    those of many."""
    rng = np.random.default_rng(21 + d)
    batch = Batch(rng, 64, [1, 40, 2, 0, 4, 5, 130], [700, 300, 0, 40, 90, 1000, 5], gap=2)
    cache = po.Pages(rng, batch.pages, 64, 2, d)
    stride = 1 << 17
    table = np.full((7, stride // 64), -1, np.int32)
    table[:, :batch.width] = batch.table
    batch.table, batch.width, batch.max_keys = table, stride // 64, 1 << 30
    assert 7 * 2 * stride * d > 64e6
    query = rng.standard_normal((batch.tokens, 8, d)).astype(np.float16 if f16 else np.float32)
    old = np.zeros((7, 2, stride), np.float32)
    old[..., :1100] = rng.random((7, 2, 1100))
    for window in (0, 3, 33):
        got = run(hip_ctx, cache, batch, 8, query, old, window, 0.8)
        want, tol = so.key_weights(cache, query, batch.plain(), 8, window, 0.8, old, stride)
        untouched = tol == 0
        assert np.array_equal(got[untouched], old[untouched])
        off = np.abs(got - want)[~untouched] / tol[~untouched]
        assert (off <= 1).all(), (window, off.max())
