"""Eviction from the paged 8-bit cache on the GPU against the plain forms
(tests/serving_oracle.py).  All outputs are equal: positions are whole numbers, and a code's
quotient, product and rounding are f32's in both."""
import math

import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_gpu_paged_q8 import DevicePages

pytestmark = pytest.mark.gpu


def run_select(ctx, weights, lengths, keep, max_keys, first, last, kept_stride):
    sequences, kv_heads, stride = weights.shape
    kept = ctx.buffer(np.full((sequences, kv_heads, kept_stride), -7, np.int32))
    out = ctx.buffer(np.full(sequences, -7, np.int32))
    ctx.select_keys_f32_i32(ctx.buffer(weights), stride, ctx.buffer(np.asarray(lengths, np.uint32)),
                            ctx.buffer(np.asarray(keep, np.uint32)), sequences, kv_heads, max_keys,
                            first, last, kept, kept_stride, out)
    return (kept.download(dtype=np.int32).reshape(sequences, kv_heads, kept_stride),
            out.download(dtype=np.uint32))


def check_select(ctx, weights, lengths, keep, first=0, last=0, max_keys=None, kept_stride=None):
    weights = np.asarray(weights, np.float32)
    max_keys = max_keys or weights.shape[2]
    kept_stride = kept_stride or max(1, max(keep))
    args = (weights, lengths, keep, max_keys, first, last, kept_stride)
    got, want = run_select(ctx, *args), so.select_keys(*args)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


def heavy(rng, *shape):
    x = np.exp(2 * rng.standard_normal(shape) - 4)
    return np.where(rng.random(shape) < 0.2, 0.0, x).astype(np.float32)


@pytest.mark.parametrize("length", [1, 2, 15, 64, 255, 1000, 1024, 1025, 4096, 5000, 33000, 70001])
def test_select_matches_plain(hip_ctx, length):
    rng = np.random.default_rng(length)
    lengths = [length, length // 2, 0, max(1, length - 1), length]
    weights = heavy(rng, 5, 2, length + 3)
    for first, last in ((0, 0), (4, 16), (1, 0), (0, 70), (length, 3), (2 ** 31, 2 ** 31)):
        keep = [max(1, length // 3), length, 3, min(length, 7), length // 2]
        check_select(hip_ctx, weights, lengths, keep, first, last, max_keys=length)


def test_select_ties_and_values_out_of_the_ordinary(hip_ctx):
    rng = np.random.default_rng(2)
    n = 3000
    rows = [np.zeros(n), np.full(n, 0.25), rng.integers(0, 3, n), np.full(n, math.nan),
            np.where(rng.random(n) < 0.5, math.nan, 1.0), np.where(rng.random(n) < 0.1, math.inf, 2),
            -rng.random(n), np.where(rng.random(n) < 0.5, -0.0, 0.0),
            rng.choice([1e-45, 0.0, 1e-40], n), rng.choice([-math.inf, math.nan, 1.0], n),
            np.arange(n), -np.arange(n), np.ldexp(1.0, rng.integers(-140, 120, n)),
            1.0 + rng.integers(0, 9, n) * 2.0 ** -23]
    weights = np.array(rows, np.float32)[:, None]
    for keep in (1, 5, 1500, 2999, 3000):
        for first, last in ((0, 0), (3, 10)):
            check_select(hip_ctx, weights, [n] * len(rows), [keep] * len(rows), first, last)


def test_select_leaves_out_what_breaks_a_bound(hip_ctx):
    rng = np.random.default_rng(3)
    weights = heavy(rng, 6, 3, 200)
    check_select(hip_ctx, weights, [150, 151, 2 ** 32 - 1, 100, 40, 150],
                 [30, 10, 5, 51, 2 ** 32 - 1, 50], 2, 4, max_keys=150, kept_stride=50)


def test_select_many_pairs(hip_ctx):
    rng = np.random.default_rng(4)
    weights = heavy(rng, 300, 5, 90)
    check_select(hip_ctx, weights, rng.integers(0, 91, 300), rng.integers(0, 60, 300), 1, 2)


def run_gather(ctx, cache, table, kept, lengths, target, weights=None, stride=0, kept_stride=None):
    pages = DevicePages(ctx, cache)
    sequences = len(table)
    bufs = [None, None]
    if weights is not None:
        bufs = [ctx.buffer(weights), ctx.buffer(np.full(weights.shape, np.nan, np.float32))]
    ctx.gather_kv_pages_q8(pages.struct, ctx.buffer(table.astype(np.int32)), table.shape[1],
                           ctx.buffer(kept.astype(np.int32)),
                           ctx.buffer(np.asarray(lengths, np.uint32)), kept_stride or kept.shape[2],
                           sequences, ctx.buffer(target.astype(np.int32)), target.shape[1],
                           bufs[0], stride, bufs[1])
    moved = None if weights is None else bufs[1].download().reshape(weights.shape)
    return pages.read(), moved


def check_gather(ctx, cache, table, kept, lengths, target, weights=None, stride=0):
    got, moved = run_gather(ctx, cache, table, kept, lengths, target, weights, stride)
    want = so.gather(cache, table, kept, lengths, kept.shape[2], target, weights, stride)
    for n in ("key", "value"):
        np.testing.assert_array_equal(got.scales[n], cache.scales[n])
        np.testing.assert_array_equal(got.codes[n], cache.codes[n])
    if weights is not None:
        np.testing.assert_array_equal(moved, want)


def scene(rng, page_tokens, kv_heads, d, source_lengths, keeps, spare=2):
    """Sequences' tables, kept positions and target pages over one pool."""
    counts = [-(-n // page_tokens) for n in source_lengths]
    targets = [-(-n // page_tokens) for n in keeps]
    pages = sum(counts) + sum(targets) + spare
    order = rng.permutation(pages)
    table = np.full((len(counts), max(counts)), -1, np.int32)
    target = np.full((len(counts), max(1, max(targets))), -1, np.int32)
    at = 0
    for rows, ns in ((table, counts), (target, targets)):
        for b, n in enumerate(ns):
            rows[b, :n] = order[at:at + n]
            at += n
    kept = np.full((len(counts), kv_heads, max(1, max(keeps))), -1, np.int32)
    for b, n in enumerate(keeps):
        for h in range(kv_heads):
            kept[b, h, :n] = np.sort(rng.permutation(source_lengths[b])[:n])
    return po.Pages(rng, pages, page_tokens, kv_heads, d), table, kept, target


@pytest.mark.parametrize("d,kv_heads", [(64, 3), (128, 8), (256, 2), (256, 1)])
@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128])
def test_gather_matches_plain(hip_ctx, d, kv_heads, page_tokens):
    rng = np.random.default_rng(d + page_tokens)
    lengths = [300, 1, 130, 57, 16]
    keeps = [120, 1, 130, 0, 9]
    cache, table, kept, target = scene(rng, page_tokens, kv_heads, d, lengths, keeps)
    weights = heavy(rng, 5, kv_heads, 310)
    check_gather(hip_ctx, cache, table, kept, keeps, target, weights, 310)


def test_gather_without_weights_and_of_equal_scales(hip_ctx):
    """Equal scales move bits."""
    rng = np.random.default_rng(5)
    cache, table, kept, target = scene(rng, 64, 2, 128, [500, 200], [77, 150])
    for n in ("key", "value"):
        cache.scales[n][:] = np.float32(0.0123)
    before = {n: cache.codes[n].copy() for n in ("key", "value")}
    check_gather(hip_ctx, cache, table, kept, [77, 150], target)
    for n in ("key", "value"):
        for h in range(2):
            j = kept[0, h, 76]
            np.testing.assert_array_equal(cache.codes[n][target[0, 1], h, 12],
                                          before[n][table[0, j // 64], h, j % 64])


def test_gather_scales_out_of_the_ordinary(hip_ctx):
    """Zero, tiny, huge and NaN scales; whole pages of zeros."""
    rng = np.random.default_rng(6)
    cache, table, kept, target = scene(rng, 16, 2, 64, [400, 400, 64], [200, 90, 40])
    values = np.array([0.0, 1e-30, 0.01, 1.0, 3e38, 1e-45, np.nan, np.inf], np.float32)
    for n in ("key", "value"):
        cache.scales[n][:] = rng.choice(values, cache.scales[n].shape,
                                        p=[.2, .1, .3, .2, .05, .1, .025, .025])
        cache.scales[n][table[2, :4]] = 0
    check_gather(hip_ctx, cache, table, kept, [200, 90, 40], target)


def test_gather_positions_and_pages_outside(hip_ctx):
    """Positions before, behind and in pages outside the pool are zeros; target pages
    outside are not written; sequences past a bound are left out."""
    rng = np.random.default_rng(7)
    cache, table, kept, target = scene(rng, 16, 2, 64, [100, 100, 100, 100], [40, 40, 40, 40])
    kept[0, 0, [0, 3, 39]] = [-1, 10 ** 6, 2 ** 31 - 1]
    kept[0, 1, 5] = -2 ** 31
    table[1, [0, 2]] = [-5, cache.pages]
    target[2, 1] = cache.pages
    target[3, 0] = -1
    weights = heavy(rng, 4, 2, 101)
    check_gather(hip_ctx, cache, table, kept, [40, 40, 40, 40], target, weights, 101)
    for lengths, stride in (([41, 40, 48, 7], 101), ([40, 2 ** 32 - 1, 0, 33], 101),
                            ([40, 12, 30, 39], 39)):
        cache, table, kept, target = scene(rng, 16, 2, 64, [100] * 4, [40] * 4)
        check_gather(hip_ctx, cache, table, kept, lengths, target,
                     np.ascontiguousarray(weights[..., :stride]), stride)


def test_gather_repeats_and_any_order(hip_ctx):
    """Positions need not rise, and one may stand twice; a source page may be shared."""
    rng = np.random.default_rng(8)
    cache, table, kept, target = scene(rng, 32, 4, 256, [90, 90], [80, 50])
    kept[0] = rng.integers(0, 90, kept[0].shape)
    table[1] = table[0]
    check_gather(hip_ctx, cache, table, kept, [80, 50], target)


def test_gather_beyond_32_bits(hip_ctx):
    """Pages whose bytes lie past 2^32 in a pool of 4.3 GiB a side."""
    torch = pytest.importorskip("torch")
    pages, pt, kv, d = 66000, 64, 4, 256
    keys = torch.zeros(pages, kv, pt, d, dtype=torch.int8, device="cuda")
    values = torch.zeros(pages, kv, pt // 8, d, 8, dtype=torch.int8, device="cuda")
    scales = [torch.full((pages, kv), 0.03, device="cuda") for _ in range(2)]
    keys[65990] = torch.randint(-127, 128, (kv, pt, d), dtype=torch.int8, device="cuda")
    values[65990] = torch.randint(-127, 128, (kv, pt // 8, d, 8), dtype=torch.int8, device="cuda")
    torch.cuda.synchronize()
    struct = kh.PagedQ8Cache(*[kh.as_buffer(t) for t in (keys, values, *scales)], pages, pt, kv, d)
    kept = np.tile(np.arange(pt, dtype=np.int32), (1, kv, 1))
    hip_ctx.gather_kv_pages_q8(struct, hip_ctx.buffer(np.array([[65990]], np.int32)), 1,
                               hip_ctx.buffer(kept), hip_ctx.buffer(np.array([pt], np.uint32)), pt, 1,
                               hip_ctx.buffer(np.array([[65999]], np.int32)), 1, None, 0, None)
    assert torch.equal(keys[65999], keys[65990]) and torch.equal(values[65999], values[65990])
    assert not bool(keys[:65990].any()) and not bool(keys[65991:65999].any())


@pytest.mark.parametrize("max_keys", [16384, 16385, 32768, 32769, 40000])
def test_select_around_what_threads_hold(hip_ctx, max_keys):
    """Lengths at and about the bounds between the forms, and a bound far above the length."""
    rng = np.random.default_rng(max_keys)
    weights = heavy(rng, 4, 1, 40000)
    check_select(hip_ctx, weights, [min(max_keys, 40000), 16384, 5000, 1], [4096, 2000, 5000, 1], 2,
                 8, max_keys=max_keys)


@pytest.mark.parametrize("page_tokens", [16, 64])
def test_captured_eviction_replays(hip_ctx, page_tokens):
    """Replays bring other weights, lengths, tables and positions; each equals the eager calls."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(page_tokens)
    n, kv, d, most, stride = 3, 2, 128, 500, 520
    width = -(-most // page_tokens)
    pages = 2 * n * width
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    names = {"keys": ((pages, kv, page_tokens, d), torch.int8),
             "values": ((pages, kv, page_tokens // 8, d, 8), torch.int8),
             "ks": ((pages, kv), torch.float32), "vs": ((pages, kv), torch.float32),
             "table": ((n, width), torch.int32), "target": ((n, width), torch.int32),
             "lengths": ((n,), torch.int32), "keep": ((n,), torch.int32),
             "w": ((n, kv, stride), torch.float32), "out": ((n, kv, stride), torch.float32),
             "kept": ((n, kv, most), torch.int32), "counts": ((n,), torch.int32)}
    sides = [{name: torch.zeros(*shape, dtype=kind, device="cuda")
              for name, (shape, kind) in names.items()} for _ in range(2)]

    def call(t):
        ctx.select_keys_f32_i32(t["w"], stride, t["lengths"], t["keep"], n, kv, most, 2, 9, t["kept"],
                                most, t["counts"])
        b = [kh.as_buffer(t[name]) for name in ("keys", "values", "ks", "vs")]
        ctx.gather_kv_pages_q8(kh.PagedQ8Cache(*b, pages, page_tokens, kv, d), t["table"], width,
                               t["kept"], t["counts"], most, n, t["target"], width, t["w"], stride,
                               t["out"])

    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(sides[0])
        for lengths, keep in (([500, 40, 0], [100, 40, 5]), ([1, 499, 300], [7, 0, 299]),
                              ([500, 500, 500], [500, 1, 250]), ([501, 64, 65], [9, 64, 1])):
            table, target = rng.permutation(pages).reshape(2, n, width)
            arrays = {"keys": rng.integers(-127, 128, names["keys"][0]),
                      "values": rng.integers(-127, 128, names["values"][0]),
                      "ks": 0.1 + rng.random((pages, kv)), "vs": 0.1 + rng.random((pages, kv)),
                      "table": table, "target": target, "lengths": np.array(lengths),
                      "keep": np.array(keep), "w": heavy(rng, n, kv, stride)}
            for t in sides:
                for name, x in arrays.items():
                    t[name].copy_(torch.from_numpy(x))
                for name in ("kept", "counts", "out"):
                    t[name].fill_(-7)
            graph.replay()
            call(sides[1])
            stream.synchronize()
            for name in names:
                assert torch.equal(sides[0][name], sides[1][name]), name
            want = so.select_keys(arrays["w"], lengths, keep, most, 2, 9, most)
            np.testing.assert_array_equal(sides[0]["kept"].cpu().numpy(), want[0])
    ctx.commit_graph()
    ctx.close()


def test_gather_leaves_pages_behind_the_kept(hip_ctx):
    """Target pages that no kept token reaches stay as they were."""
    rng = np.random.default_rng(11)
    cache, table, kept, target = scene(rng, 16, 2, 64, [100, 100, 100], [90, 17, 0], spare=20)
    spare = np.setdiff1d(np.arange(cache.pages), np.concatenate([table.ravel(), target.ravel()]))
    missing = np.argwhere(target < 0)
    target[tuple(missing.T)] = spare[:len(missing)]
    assert len(missing) > 5
    check_gather(hip_ctx, cache, table, kept, [90, 17, 0], target)
