"""Batched serving over the paged 8-bit KV cache at the edges of what its entry points
allow: bounds that are far from tight, more tiles than workgroups run at once, NaN and
infinite queries, two contexts at once, two captured graphs of one context, and the
smallest and largest rows to sample.  Tolerances are those of
tests/test_gpu_paged_q8.py and tests/test_gpu_sample.py.
"""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
from test_gpu_paged_q8 import (Batch, DevicePages, check_attention, check_pages, run_attention,
                                run_prologue)
from test_gpu_sample import check as check_sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,before", [([1, 1, 1], [9, 300, 77]), ([150], [37]),
                                        ([70, 1, 33], [5, 600, 129])])
def test_bounds_far_from_tight(hip_ctx, new, before, f16):
    """max_query and max_keys of 2^31 - 1: the launches are sized for them."""
    rng = np.random.default_rng(41)
    batch = Batch(rng, 64, new, before)
    batch.max_query = batch.max_keys = 2 ** 31 - 1
    cache = po.Pages(rng, batch.pages, 64, 2, 128)
    check_attention(hip_ctx, rng, cache, batch, 4, f16)


@pytest.mark.parametrize("sequences", [63, 64, 65, 130])
def test_many_sequences_with_chunks(hip_ctx, sequences):
    """Up to 64 sequences the workgroups choose their keys from the lengths."""
    rng = np.random.default_rng(sequences)
    new = rng.integers(0, 40, sequences)
    new[::3] = 1
    before = rng.integers(0, 700, sequences)
    batch = Batch(rng, 16, new.tolist(), before.tolist(), gap=2)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    check_attention(hip_ctx, rng, cache, batch, 6, sequences % 2 == 0)


@pytest.mark.parametrize("sequences", [1, 3])
def test_more_tiles_than_workgroups(hip_ctx, sequences):
    """9000 tokens of 32 heads in 128-row tiles: workgroups go on to further ones.  Rows
    picked at random, against the plain form of batches that hold only them."""
    rng = np.random.default_rng(43 + sequences)
    pt, kv, d, heads = 128, 2, 64, 32
    total = 9000 // sequences
    batch = Batch(rng, pt, [total - 7 * b for b in range(sequences)],
                  [40 * b for b in range(sequences)])
    cache = po.Pages(rng, batch.pages, pt, kv, d)
    query = rng.standard_normal((batch.tokens, heads, d)).astype(np.float16)
    got = run_attention(hip_ctx, cache, batch, heads, query, f16=True)
    assert not (got == -77).all(-1).any()
    for b in range(sequences):
        for i in sorted(rng.integers(0, batch.new[b], 12)) + [0, batch.new[b] - 1]:
            row = int(batch.starts[b]) + int(i)
            length = batch.before[b] + int(i) + 1
            one = (batch.table[b:b + 1], np.array([0, 1]), np.array([length]), 1, 1, length)
            want, size, score = po.attention(cache, query[row:row + 1], one, heads)
            tol = po.attention_tolerance(size, want, score, d, True)
            assert (np.abs(got[row:row + 1] - want) <= tol).all(), (b, i)


@pytest.mark.parametrize("new,before", [([1, 1], [200, 40]), ([3, 140], [40, 61])])
def test_nan_and_infinite_queries_stay_in_their_rows(hip_ctx, new, before):
    """A NaN or an infinity in a query makes its own row and head NaN or leaves them
    without meaning, and no other."""
    rng = np.random.default_rng(44)
    batch = Batch(rng, 16, new, before)
    cache = po.Pages(rng, batch.pages, 16, 2, 128)
    query = rng.standard_normal((batch.tokens, 8, 128)).astype(np.float32)
    clean = run_attention(hip_ctx, cache, batch, 8, query)
    last = batch.tokens - 1
    query[0, 3, 17] = np.nan
    query[last, 5, 0] = np.inf
    query[last, 6, 100] = -np.inf
    got = run_attention(hip_ctx, cache, batch, 8, query)
    touched = np.zeros(got.shape[:2], bool)
    touched[0, 3] = touched[last, 5] = touched[last, 6] = True
    np.testing.assert_array_equal(got[~touched], clean[~touched])
    assert np.isnan(got[0, 3]).all()


def _state(torch, seed, new, before, pt, kv, d, heads):
    rng = np.random.default_rng(seed)
    batch = Batch(rng, pt, new, before)
    cache = po.Pages(rng, batch.pages, pt, kv, d)
    t = batch.tokens
    s = {"keys": torch.from_numpy(cache.codes["key"]).cuda(),
         "values": torch.from_numpy(cache.device_values()).cuda(),
         "ks": torch.from_numpy(cache.scales["key"]).cuda(),
         "vs": torch.from_numpy(cache.scales["value"]).cuda(),
         "table": torch.from_numpy(batch.table).cuda(),
         "starts": torch.from_numpy(batch.starts.astype(np.int32)).cuda(),
         "lengths": torch.from_numpy(batch.lengths.astype(np.int32)).cuda(),
         "query": torch.from_numpy(rng.standard_normal((t, heads, d)).astype(np.float32)).cuda(),
         "out": torch.zeros(t, heads, d, device="cuda"),
         "logits": torch.from_numpy(2 * rng.standard_normal((5, 60000))).float().cuda(),
         "u": torch.from_numpy(rng.random(5).astype(np.float32)).cuda(),
         "p": torch.full((5,), 0.9, device="cuda"),
         "token": torch.zeros(5, device="cuda", dtype=torch.int32)}
    c = kh.PagedQ8Cache(*[kh.as_buffer(s[n]) for n in ("keys", "values", "ks", "vs")], batch.pages,
                        pt, kv, d)
    b = kh.PagedBatch(*[kh.as_buffer(s[n]) for n in ("table", "starts", "lengths")], len(new),
                      batch.width, t, batch.max_query, batch.max_keys)

    def step(ctx):
        ctx.attention_f32_paged_q8_kv(s["query"], None, c, b, heads, s["out"])
        ctx.sample_f32_i32(s["logits"], 5, 60000, 60000, None, None, s["p"], None, s["u"],
                           s["token"], None)

    return s, step


STATES = [(51, [1] * 9, [700 * i for i in range(9)], 64, 2, 256, 8),
          (52, [130, 1, 40], [1500, 3000, 10], 16, 4, 128, 8)]


def _results(torch, states):
    return [s[n].clone() for s, _ in states for n in ("out", "token")]


def test_two_contexts_at_once(hip_ctx):
    """Each context has its stream and workspace; steps enqueued on both side by side
    equal those of one after the other."""
    torch = pytest.importorskip("torch")
    states = [_state(torch, *a) for a in STATES]
    torch.cuda.synchronize()
    for _, step in states:
        step(hip_ctx)
    torch.cuda.synchronize()
    want = _results(torch, states)
    streams = [torch.cuda.Stream() for _ in states]
    ctxs = [kh.Context() for _ in states]
    for ctx, stream in zip(ctxs, streams):
        ctx.set_stream(stream.cuda_stream)
        ctx.begin_graph()
    for _ in range(5):
        for s, _ in states:
            s["out"].zero_()
            s["token"].zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for ctx, (_, step) in zip(ctxs, states):
                step(ctx)
        torch.cuda.synchronize()
        for x, y in zip(_results(torch, states), want):
            assert torch.equal(x, y)
    for ctx in ctxs:
        ctx.commit_graph()
        ctx.close()


def test_two_captured_graphs_of_one_context(hip_ctx):
    """Both use the context's workspace, the second after it grew; replays in turn, with
    eager work between, equal the eager results."""
    torch = pytest.importorskip("torch")
    states = [_state(torch, *a) for a in STATES]
    torch.cuda.synchronize()
    for _, step in states:
        step(hip_ctx)
    torch.cuda.synchronize()
    want = _results(torch, states)
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    ctx.begin_graph()
    graphs = []
    with torch.cuda.stream(stream):
        for _, step in states:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                step(ctx)
        for i in range(6):
            for s, _ in states:
                s["out"].zero_()
                s["token"].zero_()
            for g in graphs if i % 2 else graphs[::-1]:
                g.replay()
            stream.synchronize()
            for x, y in zip(_results(torch, states), want):
                assert torch.equal(x, y), i
            states[i % 2][1](ctx)
    ctx.commit_graph()
    ctx.close()


def test_many_short_and_one_longest_row_to_sample(hip_ctx):
    rng = np.random.default_rng(45)
    rows = 70
    check_sample(hip_ctx, np.zeros((rows, 1), np.float32), rng.random(rows).astype(np.float32),
                 top_k=[1] * rows, top_p=[0.5] * rows)
    x = (2 * rng.standard_normal((1, 4194304))).astype(np.float32)
    check_sample(hip_ctx, x, [np.float32(0.37)], top_k=[100000], top_p=[0.9])


def test_the_most_rows_to_sample(hip_ctx):
    """65535 rows, whose workspace is that of a part of them at a time."""
    rng = np.random.default_rng(46)
    rows = 65535
    x = rng.standard_normal((rows, 5)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    token, share = (hip_ctx.buffer(np.full(rows, -7, np.int32)), hip_ctx.buffer(
        np.full(rows, -7, np.float32)))
    hip_ctx.sample_f32_i32(hip_ctx.buffer(x), rows, 5, 5, None, None, None, None,
                           hip_ctx.buffer(u), token, share)
    w = np.exp(x.astype(np.float64) - x.max(1, keepdims=True))
    run = np.cumsum(w, 1) / w.sum(1, keepdims=True)
    clear = np.abs(run - u[:, None]).min(1) > 1e-9
    want = (run <= u[:, None]).sum(1)
    got = token.download(dtype=np.int32)
    np.testing.assert_array_equal(got[clear], want[clear])
    assert clear.mean() > 0.999
    p = (w / w.sum(1, keepdims=True))[np.arange(rows), got]
    assert (np.abs(share.download() - p) <= 2.0 ** -23 * p).all()


def test_pages_read_back_twice(hip_ctx):
    """The same page id more than once, and ids outside the pool between."""
    rng = np.random.default_rng(47)
    cache = po.Pages(rng, 5, 32, 3, 64)
    pages = DevicePages(hip_ctx, cache)
    ids = np.array([3, 3, -1, 0, 5, 3], np.int32)
    rows = [hip_ctx.buffer(np.full(6 * 32 * 3 * 64, 9, np.float16)) for _ in range(2)]
    hip_ctx.dequantize_kv_pages_q8_f16(pages.struct, hip_ctx.buffer(ids), 6, *rows)
    for r, n in zip(rows, ("key", "value")):
        got = r.download(dtype=np.float16).reshape(6, 32, 3, 64)
        for i, page in enumerate(ids):
            want = (cache.values_of(n, page).astype(np.float32).astype(np.float16)
                    if 0 <= page < 5 else np.zeros((32, 3, 64), np.float16))
            np.testing.assert_array_equal(got[i], want)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,before", [([4, 1, 2, 0, 3], [9, 300, 1000, 5, 0]), ([4], [700]),
                                        ([3], [40]), ([2, 9, 4], [129, 64, 500])])
def test_blocks_of_rows(hip_ctx, new, before, f16):
    """17 to 32 rows of a sequence and KV head, more than one block of the decode kernel,
    alone and beside shorter and longer ones."""
    rng = np.random.default_rng(48)
    batch = Batch(rng, 32, new, before, gap=1)
    for heads, kv, d in ((14, 2, 64), (8, 1, 128), (24, 3, 256)):
        cache = po.Pages(rng, batch.pages, 32, kv, d)
        check_attention(hip_ctx, rng, cache, batch, heads, f16, gated=not f16)


@pytest.mark.parametrize("cluster", [2, 63, 64, 65, 129, 700])
def test_cuts_inside_clusters(hip_ctx, cluster):
    """Logits within a few steps of each other, many of them equal, and cuts among them:
    a threshold's last digits hold one, few and many entries."""
    rng = np.random.default_rng(cluster)
    rows, size = 12, 9000
    x = (rng.standard_normal((rows, size)) - 4).astype(np.float32)
    for r in range(rows):
        at = rng.permutation(size)[:cluster]
        x[r, at] = np.float32(2.0) + rng.integers(0, 1 + r * cluster // 8, cluster).astype(
            np.float32) * np.float32(2.0 ** -22)
        x[r, rng.permutation(size)[:3]] = 3.0
    u = rng.random(rows).astype(np.float32)
    k = np.clip(rng.integers(1, cluster + 8, rows), 1, size).astype(np.int32)
    check_sample(hip_ctx, x, u, top_k=k.tolist())
    check_sample(hip_ctx, x, u, top_p=rng.uniform(0.05, 0.6, rows).astype(np.float32).tolist())
    check_sample(hip_ctx, x, u, top_k=k.tolist(), top_p=[0.5] * rows)


@pytest.mark.parametrize("page_tokens,new,before", [
    (32, [20, 1, 90], [3, 31, 64]), (128, [200, 1, 60], [40, 127, 256]), (128, [20], [120]),
    (64, [30, 64], [50, 0]), (16, [3, 4], [14, 31])])
def test_prologue_rows_per_page(hip_ctx, page_tokens, new, before):
    """Every number of waves that a page's rows are spread over."""
    rng = np.random.default_rng(page_tokens + len(new))
    batch = Batch(rng, page_tokens, new, before, gap=1)
    for heads, kv, d in ((6, 3, 64), (8, 2, 256)):
        cache = po.Pages(rng, batch.pages, page_tokens, kv, d)
        q, gate, got_q, got_gate, pages, exact = run_prologue(hip_ctx, rng, cache, batch, heads, 64,
                                                              (11, 11, 10, 0))
        check_pages(cache, pages.read(), exact)
        step = np.abs(q[:batch.rows]).max(-1, keepdims=True) * 2.0 ** -19
        assert (np.abs(got_q - q)[:batch.rows] <= step).all()
        np.testing.assert_array_equal(got_gate[:batch.rows], gate[:batch.rows])
        assert (got_q[batch.rows:] == -77).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,before", [([1], [300]), ([1, 1, 3], [40, 900, 0])])
def test_more_query_heads_than_a_block(hip_ctx, new, before, f16):
    """40 query heads of one KV head: one token is more than 32 rows."""
    rng = np.random.default_rng(49)
    batch = Batch(rng, 64, new, before)
    cache = po.Pages(rng, batch.pages, 64, 1, 64)
    check_attention(hip_ctx, rng, cache, batch, 40, f16)
