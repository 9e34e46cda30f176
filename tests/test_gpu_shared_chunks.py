"""Prompt chunks behind a shared prefix, on the GPU: where the sequences' rows fill tiles by
themselves the shared entry makes the plain call, bit by bit; beside many single tokens it shares,
eager and in captured steps."""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_gpu_paged_q8 import HEADS, Batch, DevicePages
from test_gpu_shared_prefix import check, run

pytestmark = pytest.mark.gpu


def plain(ctx, cache, batch, heads, query, max_keys):
    pages, tables = DevicePages(ctx, cache), batch.device(ctx)
    tables.max_keys = max_keys
    out = ctx.buffer(np.full(query.shape, -77.0, query.dtype))
    q = ctx.buffer(query)
    if query.dtype == np.float16:
        ctx.attention_f16q_paged_q8_kv(q, pages.struct, tables, heads, out)
    else:
        ctx.attention_f32_paged_q8_kv(q, None, pages.struct, tables, heads, out)
    return out.download(dtype=query.dtype).reshape(query.shape).astype(np.float64)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,heads", [([100, 90, 110], 8), ([64] * 6, 4), ([256, 1, 1], 4),
                                       ([512, 300], 2)])
def test_chunks_that_fill_tiles_take_the_plain_call(hip_ctx, new, heads, f16):
    rng = np.random.default_rng(len(new))
    batch = Batch(rng, 16, new, [320 + 7 * i for i in range(len(new))])
    cache = po.Pages(rng, batch.pages, 16, 2, 128)
    assert batch.tokens * heads // 2 >= 128 * len(new)
    groups = so.share_prefixes(16, batch, [(0, len(new), 320)])
    query = rng.standard_normal((batch.tokens, heads, 128)).astype(np.float16 if f16 else np.float32)
    got = run(hip_ctx, cache, batch, groups, heads, query)
    np.testing.assert_array_equal(got, plain(hip_ctx, cache, batch, heads, query, 1 << 20))
    check(hip_ctx, rng, cache, batch, groups, heads, f16)


# Chunks beside single tokens and drafted ones, few enough rows at the mean to share.
MIXED = ([40, 1, 90, 2, 1, 1, 0, 8, 1, 33, 1, 1],
         [128, 500, 130, 140, 300, 129, 128, 260, 700, 128, 190, 131])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("d,heads,kv_heads", [*HEADS, (64, 4, 1)])
def test_chunks_beside_single_tokens_share(hip_ctx, d, heads, kv_heads, page_tokens, f16):
    rng = np.random.default_rng(d + heads + page_tokens)
    batch = Batch(rng, page_tokens, *MIXED, gap=2)
    assert batch.tokens * heads // kv_heads < 128 * len(batch.new)
    cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
    for shared in ([(0, 12, 128)], [(0, 3, 128), (4, 12, 128)]):
        groups = so.share_prefixes(page_tokens, batch, shared)
        check(hip_ctx, rng, cache, batch, groups, heads, f16, gated=not f16)


@pytest.mark.parametrize("f16", [False, True])
def test_captured_step_with_chunks_replays(hip_ctx, f16):
    """Replays bring other chunks, groups and prefixes in the same arrays; each equals the
    eager call bit by bit, and the plain form to its tolerance."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(31)
    d, heads, kv, pt, n, width, tokens = 128, 8, 2, 16, 8, 60, 150
    cache = po.Pages(rng, n * width + 20, pt, kv, d)
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
    pages = kh.PagedQ8Cache(v["keys"], v["values"], v["ks"], v["vs"], cache.pages, pt, kv, d)
    batch = kh.PagedBatch(v["table"], v["starts"], v["lengths"], n, width, tokens, 100, 1 << 20)
    prefixes = kh.SharedPrefixes(v["gs"], v["gl"], 2, tokens, 1 << 20)
    assert tokens * heads // kv < 128 * n

    def call(out):
        if f16:
            ctx.attention_f16q_shared_paged_q8_kv(v["q"], pages, batch, prefixes, heads, v[out])
        else:
            ctx.attention_f32_shared_paged_q8_kv(v["q"], None, pages, batch, prefixes, heads,
                                                 v[out])

    sets = [([100, 1, 1, 1, 30, 1, 1, 1], [640, 700, 650, 800, 641, 643, 640, 700], [(0, 8, 640)]),
            ([1] * 8, [400, 450, 399, 390, 100, 90, 85, 80], [(0, 4, 384), (4, 8, 80)]),
            ([3, 0, 9, 1, 17, 33, 1, 64], [10, 20, 900, 830, 5, 850, 800, 805],
             [(5, 8, 800)]),
            ([1, 90, 1, 1, 40, 1, 1, 1], [3, 5, 7, 9, 20, 30, 40, 50], [(0, 8, 0)])]
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph, out in zip(graphs, ("a", "c")):
            with torch.cuda.graph(graph, stream=stream):
                call(out)
        for new, before, shared in sets:
            host = Batch(rng, pt, new, before)
            host.table = rng.permutation(n * width).reshape(n, width).astype(np.int32)
            starts, lengths = so.share_prefixes(pt, host, shared)
            gs, gl = np.full(3, n), np.zeros(2)
            gs[:len(starts)], gl[:len(lengths)] = starts, lengths
            for name, x in (("table", host.table), ("starts", host.starts.astype(np.int32)),
                            ("lengths", host.lengths.astype(np.int32)), ("gs", gs.astype(np.int32)),
                            ("gl", gl.astype(np.int32)),
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
