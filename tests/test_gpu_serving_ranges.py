"""Key weights and shared prefixes in pools past 2^32 bytes, and the serving entries on two
streams at once."""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_gpu_paged_q8 import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [40, 1]])
def test_pages_beyond_32_bits(hip_ctx, new, f16):
    """The same bits from pages at the end of a pool of 4.3 GiB a side as from a small one."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(30 + sum(new))
    pt, kv, d, heads, far = 64, 4, 256, 8, 66000
    batch = Batch(rng, pt, new, [900, 1000])
    groups = so.share_prefixes(pt, batch, [(0, 2, 896)])
    cache = po.Pages(rng, batch.pages, pt, kv, d)
    kind = np.float16 if f16 else np.float32
    query = hip_ctx.buffer(rng.standard_normal((batch.tokens, heads, d)).astype(kind))
    gs, gl = (hip_ctx.buffer(np.asarray(x, np.uint32)) for x in groups)
    prefixes = kh.SharedPrefixes(gs.view, gl.view, 1, batch.tokens, 1 << 40)
    base = far - cache.pages
    found = []
    for shift, pages in ((0, cache.pages), (base, far)):
        t = [torch.zeros(pages, kv, pt, d, dtype=torch.int8, device="cuda"),
             torch.zeros(pages, kv, pt // 8, d, 8, dtype=torch.int8, device="cuda"),
             torch.full((pages, kv), 0.5, device="cuda"), torch.full((pages, kv), 0.5, device="cuda")]
        for x, host in zip(t, (cache.codes["key"], cache.device_values(), cache.scales["key"],
                               cache.scales["value"])):
            x[shift:] = torch.from_numpy(host).cuda()
        torch.cuda.synchronize()
        struct = kh.PagedQ8Cache(*[kh.as_buffer(x) for x in t], pages, pt, kv, d)
        small = batch.table
        batch.table = np.where(small < 0, small, small + shift).astype(np.int32)
        tables = batch.device(hip_ctx)
        tables.max_keys = 1 << 20
        batch.table = small
        out = hip_ctx.buffer(np.zeros((batch.tokens, heads, d), kind))
        weights = hip_ctx.buffer(np.zeros((2, kv, 1100), np.float32))
        if f16:
            hip_ctx.attention_f16q_shared_paged_q8_kv(query, struct, tables, prefixes, heads, out)
            hip_ctx.key_weights_f16q_paged_q8_kv(query, struct, tables, heads, 0, 0.0, weights, 1100)
        else:
            hip_ctx.attention_f32_shared_paged_q8_kv(query, None, struct, tables, prefixes, heads, out)
            hip_ctx.key_weights_f32_paged_q8_kv(query, struct, tables, heads, 0, 0.0, weights, 1100)
        found.append((out.download(dtype=kind), weights.download()))
        del t
    np.testing.assert_array_equal(found[0][0], found[1][0])
    np.testing.assert_array_equal(found[0][1], found[1][1])
    sums = found[0][1].reshape(2, kv, 1100).sum(-1)
    np.testing.assert_allclose(sums, 2.0 * np.array(new)[:, None] * np.ones((1, kv)), rtol=1e-5)


def test_two_contexts_at_once(hip_ctx):
    """Calls of two contexts, each with its stream and workspace, that run side by side."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(33)
    pt, kv, d, heads, stride = 16, 2, 128, 8, 1500
    sides = []
    for new, before in (([1] * 6, [1000, 900, 880, 1200, 870, 1400]), ([70, 3, 1], [800, 600, 900])):
        batch = Batch(rng, pt, new, before)
        n = len(new)
        groups = so.share_prefixes(pt, batch, [(0, n, 592)])
        cache = po.Pages(rng, batch.pages, pt, kv, d)
        size = 30000 + 700 * n
        host = {"keys": cache.codes["key"], "values": cache.device_values(),
                "ks": cache.scales["key"], "vs": cache.scales["value"], "table": batch.table,
                "starts": batch.starts.astype(np.int32), "lengths": batch.lengths.astype(np.int32),
                "gs": groups[0].astype(np.int32), "gl": groups[1].astype(np.int32),
                "q": rng.standard_normal((batch.tokens, heads, d)).astype(np.float32),
                "out": np.zeros((batch.tokens, heads, d), np.float32),
                "w": np.zeros((n, kv, stride), np.float32), "keep": np.full(n, 200, np.int32),
                "kept": np.zeros((n, kv, 200), np.int32), "counts": np.zeros(n, np.int32),
                "logits": (3 * rng.standard_normal((n, size))).astype(np.float32),
                "entropy": np.zeros(n, np.float32), "top": np.zeros((n, 20), np.int32)}
        t = {name: torch.from_numpy(np.ascontiguousarray(x)).cuda() for name, x in host.items()}
        b = {name: kh.as_buffer(x) for name, x in t.items()}
        stream, ctx = torch.cuda.Stream(), kh.Context()
        ctx.set_stream(stream.cuda_stream)
        sides.append((ctx, stream, t, b, kh.PagedQ8Cache(b["keys"], b["values"], b["ks"], b["vs"],
                                                         cache.pages, pt, kv, d),
                      kh.PagedBatch(b["table"], b["starts"], b["lengths"], n, batch.width,
                                    batch.tokens, batch.max_query, 1 << 20),
                      kh.SharedPrefixes(b["gs"], b["gl"], 1, batch.tokens, 1 << 20), n, size))

    def call(side):
        ctx, _, t, b, pages, batch, groups, n, size = side
        ctx.attention_f32_shared_paged_q8_kv(b["q"], None, pages, batch, groups, heads, b["out"])
        ctx.key_weights_f32_paged_q8_kv(b["q"], pages, batch, heads, 0, 0.0, b["w"], stride)
        ctx.select_keys_f32_i32(b["w"], stride, b["lengths"], b["keep"], n, kv, stride, 4, 16, b["kept"],
                                200, b["counts"])
        ctx.token_logprobs_f32(b["logits"], n, size, size, None, None, 20, None, None, b["entropy"],
                               b["top"], None)

    names = ("out", "w", "kept", "counts", "entropy", "top")
    torch.cuda.synchronize()
    alone = []
    for side in sides:
        side[0].begin_graph()
        call(side)
        side[1].synchronize()
        alone.append({name: side[2][name].clone() for name in names})
    torch.cuda.synchronize()
    for _ in range(10):
        for side in sides:
            with torch.cuda.stream(side[1]):
                for name in names:
                    side[2][name].zero_()
            call(side)
        for side, want in zip(sides, alone):
            side[1].synchronize()
            for name in names:
                assert torch.equal(side[2][name], want[name]), name
    for side in sides:
        side[0].commit_graph()
        side[0].close()
