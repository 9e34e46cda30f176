"""Attention of batches whose sequences share prefixes, on the GPU: the outputs of the
plain form of attention (tests/paged_oracle.py) to its tolerance, whose 64 half steps for
sums cover the join of a prefix's part with the rest (a few roundings).

Where the bounds promise little to share the library takes the plain call; the tests
loosen them so that these small batches share."""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_gpu_paged_q8 import HEADS, Batch, DevicePages

pytestmark = pytest.mark.gpu


def run(ctx, cache, batch, groups, heads, query, gate=None, max_rows=None, max_prefix=None,
        loose=True):
    starts, lengths = groups
    pages, tables = DevicePages(ctx, cache), batch.device(ctx)
    if loose and max_prefix is None:
        max_prefix = 2 ** 40
    keep = [ctx.buffer(np.asarray(starts, np.uint32)), ctx.buffer(np.asarray(lengths, np.uint32))]
    prefixes = kh.SharedPrefixes(*[b.view for b in keep], len(lengths), max_rows or batch.tokens,
                                 max_prefix or max(1, int(max(lengths))))
    if loose and batch.max_keys == max(1, int(batch.lengths.max())):
        tables.max_keys = 1 << 20
    out = ctx.buffer(np.full(query.shape, -77.0, query.dtype))
    q = ctx.buffer(query)
    if query.dtype == np.float16:
        ctx.attention_f16q_shared_paged_q8_kv(q, pages.struct, tables, prefixes, heads, out)
    else:
        g = None if gate is None else ctx.buffer(gate)
        ctx.attention_f32_shared_paged_q8_kv(q, g, pages.struct, tables, prefixes, heads, out)
    return out.download(dtype=query.dtype).reshape(query.shape).astype(np.float64)


def check(ctx, rng, cache, batch, groups, heads, f16, gated=False, **bounds):
    kind = np.float16 if f16 else np.float32
    query = (2.0 * rng.standard_normal((batch.tokens, heads, cache.head_dim))).astype(kind)
    gate = rng.standard_normal(query.shape).astype(np.float32) if gated else None
    got = run(ctx, cache, batch, groups, heads, query, gate, **bounds)
    want, size, score = po.attention(cache, query, batch.plain(), heads, gate)
    rows = ~np.isnan(size[..., 0])
    tol = po.attention_tolerance(size, want, score, cache.head_dim, f16)
    assert (got[~rows] == -77).all()
    off = np.abs(got - want)[rows] / tol[rows]
    assert (off <= 1).all(), (off.max(), np.argwhere(~(off <= 1))[:4])
    return got


# (new tokens, tokens before) of the sequences, (first, end, prefix) of the groups.
MIXES = {
    "pair": ([1, 1], [70, 64], [(0, 2, 64)]),
    "decode": ([1] * 9, [200, 130, 128, 129, 400, 128, 191, 192, 700], [(0, 9, 128)]),
    "two groups": ([1, 1, 1, 1, 1, 1], [64, 99, 300, 310, 290, 5], [(0, 2, 64), (2, 5, 288)]),
    "verify": ([8, 8, 5, 1], [260, 300, 256, 900], [(0, 4, 256)]),
    "with chunks": ([40, 1, 90, 2], [128, 500, 130, 140], [(0, 4, 128)]),
    "among others": ([1, 30, 1, 1, 0, 1], [10, 0, 333, 400, 321, 900], [(2, 6, 320)]),
    "one of one": ([1, 1], [500, 600], [(0, 1, 448), (1, 2, 576)]),
    "whole before": ([3, 2, 1], [128, 128, 128], [(0, 3, 128)]),
}


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("d,heads,kv_heads", HEADS)
def test_matches_plain(hip_ctx, d, heads, kv_heads, page_tokens, mix, f16):
    rng = np.random.default_rng(d + heads + page_tokens)
    new, before, shared = MIXES[mix]
    batch = Batch(rng, page_tokens, new, before, gap=2)
    cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
    groups = so.share_prefixes(page_tokens, batch, shared)
    for loose in (True, False):
        check(hip_ctx, rng, cache, batch, groups, heads, f16, gated=not f16, loose=loose)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("members,new,prefix,d,heads,kv_heads", [
    (40, 1, 3000, 256, 8, 2), (5, 1, 20000, 256, 8, 2), (3, 1, 6000, 64, 24, 2),
    (30, 6, 2500, 128, 16, 8), (70, 1, 1500, 128, 4, 1), (2, 150, 4000, 256, 4, 1)])
def test_long_prefixes(hip_ctx, members, new, prefix, d, heads, kv_heads, f16):
    rng = np.random.default_rng(prefix)
    own = rng.integers(0, 400, members)
    batch = Batch(rng, 64, [new] * members, (prefix // 64 * 64 + own).tolist())
    cache = po.Pages(rng, batch.pages, 64, kv_heads, d)
    groups = so.share_prefixes(64, batch, [(0, members, prefix)])
    for loose in (True, False):
        check(hip_ctx, rng, cache, batch, groups, heads, f16, loose=loose)


@pytest.mark.parametrize("f16", [False, True])
def test_prefixes_that_count_in_part(hip_ctx, f16):
    """Not whole pages, longer than what a member has before its new tokens (its tables
    then begin alike as far only), none at all, shorter than a page."""
    rng = np.random.default_rng(21)
    for prefix in (1, 15, 16, 50, 100, 300):
        batch = Batch(rng, 16, [1, 2, 40, 0, 1], [200, 61, 90, 7, 150])
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        groups = so.share_prefixes(16, batch, [(0, 5, prefix)])
        check(hip_ctx, rng, cache, batch, groups, 6, f16)
    batch = Batch(rng, 16, [1, 1], [40, 0])
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    check(hip_ctx, rng, cache, batch, so.share_prefixes(16, batch, [(0, 2, 32)]), 6, f16)


@pytest.mark.parametrize("f16", [False, True])
def test_groups_that_break_a_bound_share_nothing(hip_ctx, f16):
    rng = np.random.default_rng(22)
    new, before = [1, 2, 1, 3, 1, 1], [100, 90, 200, 64, 70, 300]
    batch = Batch(rng, 16, new, before, gap=1)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    so.share_prefixes(16, batch, [(0, 3, 80), (3, 6, 64)])
    for starts, lengths, bounds in (
            ([0, 3, 6], [80, 64], dict(max_rows=4)),
            ([0, 3, 6], [80, 64], dict(max_rows=3)),
            ([0, 3, 6], [80, 64], dict(max_prefix=79)),
            ([0, 3, 7], [80, 64], {}), ([0, 3, 2 ** 32 - 1], [80, 64], {}),
            ([3, 0, 6], [64, 0], {}), ([7, 3, 6], [64, 64], {}),
            ([6, 6, 6], [80, 64], {}), ([0, 3, 6], [2 ** 32 - 1, 64], dict(max_prefix=100)),
            ([0, 0, 0, 3, 3, 6, 6], [9, 9, 80, 7, 64, 9], {})):
        check(hip_ctx, rng, cache, batch, (starts, lengths), 4, f16, **bounds)


@pytest.mark.parametrize("spoil", ["length", "query", "width", "starts"])
def test_sequences_that_break_a_bound(hip_ctx, spoil):
    """A member that is left out: nothing of it is written, the others have their keys."""
    rng = np.random.default_rng(23)
    for f16 in (False, True):
        batch = Batch(rng, 16, [1, 12, 1, 3], [100, 200, 90, 85], gap=1)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        groups = so.share_prefixes(16, batch, [(0, 4, 80)])
        if spoil == "length":
            batch.max_keys = 150
        elif spoil == "query":
            batch.max_query = 8
        elif spoil == "width":
            batch.lengths[1] = 16 * batch.width + 1
            batch.max_keys = 1000
        else:
            batch.starts[2] = 14  # the third sequence has no rows, the second too many
            batch.starts[3] = 14
            batch.max_query = 12
        check(hip_ctx, rng, cache, batch, groups, 4, f16)


@pytest.mark.parametrize("f16", [False, True])
def test_pages_outside_and_scales_out_of_the_ordinary(hip_ctx, f16):
    """Prefix pages outside the pool, all of a prefix outside, zero scales, and a NaN that
    stays with the group and KV head that use it."""
    rng = np.random.default_rng(24)
    batch = Batch(rng, 16, [1, 1, 30, 1, 1], [100, 130, 96, 64, 70])
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    groups = so.share_prefixes(16, batch, [(0, 3, 96), (3, 5, 64)])
    for b in range(3):
        batch.table[b, [1, 4]] = [-1, cache.pages]
    for b in (3, 4):
        batch.table[b, :4] = 2 ** 31 - 1
    cache.scales["value"][batch.table[0, 2]] = 0.0
    cache.scales["key"][batch.table[0, 3]] = 0.0
    check(hip_ctx, rng, cache, batch, groups, 6, f16)
    query = rng.standard_normal((batch.tokens, 6, 64)).astype(np.float16 if f16 else np.float32)
    want = run(hip_ctx, cache, batch, groups, 6, query)
    for name in ("key", "value"):
        held = cache.scales[name][batch.table[0, 0], 1]
        cache.scales[name][batch.table[0, 0], 1] = np.nan
        got = run(hip_ctx, cache, batch, groups, 6, query)
        assert np.isnan(got[:32, 3:]).all()
        np.testing.assert_array_equal(got[:, :3], want[:, :3])
        np.testing.assert_array_equal(got[32:], want[32:])
        cache.scales[name][batch.table[0, 0], 1] = held
    spoiled = query.copy()
    spoiled[1, 2, 7] = np.nan
    got = run(hip_ctx, cache, batch, groups, 6, spoiled)
    assert np.isnan(got[1, 2]).all()
    rest = np.ones(got.shape[:2], bool)
    rest[1, 2] = False
    np.testing.assert_array_equal(got[rest], want[rest])


@pytest.mark.parametrize("f16", [False, True])
def test_bounds_far_from_tight(hip_ctx, f16):
    rng = np.random.default_rng(25)
    new, before, shared = MIXES["verify"]
    for spread in (new, [1, 1, 1, 1]):
        batch = Batch(rng, 64, spread, before)
        batch.max_query = batch.max_keys = 2 ** 31 - 1
        cache = po.Pages(rng, batch.pages, 64, 2, 128)
        groups = so.share_prefixes(64, batch, shared)
        check(hip_ctx, rng, cache, batch, groups, 4, f16, max_rows=2 ** 40, max_prefix=2 ** 40)


@pytest.mark.parametrize("sequences", [64, 65, 150])
def test_many_groups_and_sequences(hip_ctx, sequences):
    rng = np.random.default_rng(sequences)
    new = rng.integers(0, 6, sequences)
    before = (rng.integers(3, 30, sequences) * 16 + rng.integers(0, 16, sequences))
    batch = Batch(rng, 16, new.tolist(), before.tolist(), gap=2)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    shared, at = [], 0
    while at < sequences:
        n = min(int(rng.integers(1, 9)), sequences - at)
        shared.append((at, at + n, int(min(before[at:at + n]))))
        at += n
    groups = so.share_prefixes(16, batch, shared)
    check(hip_ctx, rng, cache, batch, groups, 6, sequences % 2 == 0)


@pytest.mark.parametrize("f16", [False, True])
def test_hundreds_of_pairs_some_past_the_bound(hip_ctx, f16):
    """More items than the plan holds on the chip, tight bounds, prefixes above max_prefix."""
    rng = np.random.default_rng(27)
    sequences = 800
    before = rng.integers(0, 500, sequences)
    batch = Batch(rng, 16, [1] * sequences, before.tolist())
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    shared = [(b, b + 2, int(rng.integers(0, 600))) for b in range(0, sequences, 2)]
    groups = so.share_prefixes(16, batch, shared)
    check(hip_ctx, rng, cache, batch, groups, 4, f16, max_prefix=400, max_rows=2, loose=False)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,heads,kv_heads,page_tokens", [(256, 16, 1, 32), (128, 5, 5, 128),
                                                         (64, 24, 2, 128), (128, 34, 2, 32)])
def test_group_sizes(hip_ctx, d, heads, kv_heads, page_tokens, f16):
    rng = np.random.default_rng(d + heads)
    for new, before in (([1, 1, 1], [400, 384, 900]), ([9, 1, 70], [390, 700, 500])):
        batch = Batch(rng, page_tokens, new, before)
        cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
        groups = so.share_prefixes(page_tokens, batch, [(0, 3, 384)])
        check(hip_ctx, rng, cache, batch, groups, heads, f16)


@pytest.mark.parametrize("f16", [False, True])
def test_captured_step_replays_with_other_groups(hip_ctx, f16):
    """Replays bring other lengths, groups and prefixes in the same arrays; each equals the
    eager call bit by bit, and what a second graph of the context ran between."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(26)
    d, heads, kv, pt, n, width, tokens = 128, 8, 2, 16, 4, 60, 130
    cache = po.Pages(rng, 260, pt, kv, d)
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    kind = torch.float16 if f16 else torch.float32
    t = {"keys": torch.from_numpy(cache.codes["key"]).cuda(),
         "values": torch.from_numpy(cache.device_values()).cuda(),
         "ks": torch.from_numpy(cache.scales["key"]).cuda(),
         "vs": torch.from_numpy(cache.scales["value"]).cuda(),
         "table": torch.zeros(n, width, dtype=torch.int32, device="cuda"),
         "starts": torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
         "lengths": torch.zeros(n, dtype=torch.int32, device="cuda"),
         "gs": torch.zeros(3, dtype=torch.int32, device="cuda"),
         "gl": torch.zeros(2, dtype=torch.int32, device="cuda")}
    for name in ("q", "a", "b", "c"):
        t[name] = torch.zeros(tokens, heads, d, device="cuda", dtype=kind)
    v = {name: kh.as_buffer(x) for name, x in t.items()}
    pages = kh.PagedQ8Cache(v["keys"], v["values"], v["ks"], v["vs"], 260, pt, kv, d)
    batch = kh.PagedBatch(v["table"], v["starts"], v["lengths"], n, width, tokens, 100, 1 << 20)
    prefixes = kh.SharedPrefixes(v["gs"], v["gl"], 2, tokens, 1 << 20)

    def call(out):
        if f16:
            ctx.attention_f16q_shared_paged_q8_kv(v["q"], pages, batch, prefixes, heads, v[out])
        else:
            ctx.attention_f32_shared_paged_q8_kv(v["q"], None, pages, batch, prefixes, heads,
                                                 v[out])

    sets = [([1, 1, 1, 1], [800, 850, 900, 803], [(0, 4, 800)]),
            ([1, 1, 1, 1], [400, 450, 100, 90], [(0, 2, 384), (2, 4, 80)]),
            ([100, 4, 1, 20], [640, 700, 650, 800], [(0, 4, 640)]),
            ([2, 0, 1, 1], [10, 20, 900, 900], [(2, 4, 880)]),
            ([1, 90, 1, 1], [3, 5, 7, 9], [(0, 4, 0)])]
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph, out in zip(graphs, ("a", "c")):
            with torch.cuda.graph(graph, stream=stream):
                call(out)
        for new, before, shared in sets:
            host = Batch(rng, pt, new, before)
            host.table = rng.permutation(260)[:n * width].reshape(n, width).astype(np.int32)
            starts, lengths = so.share_prefixes(pt, host, shared)
            starts = np.concatenate([starts, [n] * (3 - len(starts))])
            lengths = np.concatenate([lengths, [0] * (2 - len(lengths))])
            for name, x in (("table", host.table), ("starts", host.starts.astype(np.int32)),
                            ("lengths", host.lengths.astype(np.int32)),
                            ("gs", starts.astype(np.int32)), ("gl", lengths.astype(np.int32)),
                            ("q", rng.standard_normal((tokens, heads, d)).astype(
                                np.float16 if f16 else np.float32))):
                t[name].copy_(torch.from_numpy(x))
            for name in ("a", "b", "c"):
                t[name].fill_(-77)
            graphs[0].replay()
            call("b")
            graphs[1].replay()
            stream.synchronize()
            assert torch.equal(t["a"], t["b"]) and torch.equal(t["a"], t["c"])
            assert bool((t["a"][host.rows:] == -77).all())
            host.tokens, host.max_query, host.max_keys, host.width = tokens, 100, 1 << 20, width
            query = t["q"].cpu().numpy()
            want, size, score = po.attention(cache, query, host.plain(), heads)
            tol = po.attention_tolerance(size, want, score, d, f16)
            rows = ~np.isnan(size[..., 0])
            got = t["a"].cpu().numpy().astype(np.float64)
            assert (np.abs(got - want)[rows] <= tol[rows]).all()
    ctx.commit_graph()
    ctx.close()
