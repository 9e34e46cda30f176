"""The paged 8-bit KV cache on the GPU against plain 64-bit forms
(tests/paged_oracle.py): the attention prologue into pages, attention over them and
pages read back.

Tolerances, from the roundings counted in half steps of f32 (2^-24):
- query_out: the norm's sum, division and square root, two products and a rotation
  are under 16 of them relative to the head's largest normed value, and the
  angle's fraction of a turn is off by 2^-25 of one (pi 2^-24): 2^-19 of that value.
- codes: equal, except where the value over its scale lies within 127 * 2^-19 of the
  border of two codes; scales: the largest value's error, 2^-19.
- attention: paged_oracle.attention_tolerance.
"""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po

pytestmark = pytest.mark.gpu

THETA, EPS = 1e7, 1e-6


class Batch:
    """Tables of a batch over random pages, with `spare` pages that no sequence has."""

    def __init__(self, rng, page_tokens, new, before, spare=2, gap=0):
        self.new, self.before = list(new), list(before)
        self.lengths = np.array([a + b for a, b in zip(new, before)], np.uint32)
        counts = [-(-int(l) // page_tokens) for l in self.lengths]
        self.pages = max(1, sum(counts)) + spare
        self.width = max(1, max(counts))
        order = rng.permutation(self.pages)
        self.table = np.full((len(new), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.rows = int(self.starts[-1])
        self.tokens = self.rows + gap
        self.max_query = max(1, max(new))
        self.max_keys = max(1, int(self.lengths.max()))

    def plain(self):
        return (self.table, self.starts.astype(np.int64), self.lengths.astype(np.int64),
                self.tokens, self.max_query, self.max_keys)

    def device(self, ctx):
        self.keep = [ctx.buffer(self.table), ctx.buffer(self.starts), ctx.buffer(self.lengths)]
        return kh.PagedBatch(*[b.view for b in self.keep], len(self.new), self.width, self.tokens,
                             self.max_query, self.max_keys)


class DevicePages:
    def __init__(self, ctx, cache):
        self.cache = cache
        self.keep = [ctx.buffer(cache.codes["key"]), ctx.buffer(cache.device_values()),
                     ctx.buffer(cache.scales["key"]), ctx.buffer(cache.scales["value"])]
        self.struct = kh.PagedQ8Cache(*[b.view for b in self.keep], cache.pages,
                                      cache.page_tokens, cache.kv_heads, cache.head_dim)

    def read(self):
        """A Pages object with what the device holds."""
        out = po.Pages.__new__(po.Pages)
        out.__dict__.update(self.cache.__dict__)
        shape = self.cache.codes["key"].shape
        out.codes = {"key": self.keep[0].download(dtype=np.int8).reshape(shape)}
        out.codes["value"] = np.empty(shape, np.int8)
        out.set_device_values(self.keep[1].download(dtype=np.int8))
        out.scales = {n: self.keep[i].download(dtype=np.float32).reshape(shape[:2])
                      for n, i in (("key", 2), ("value", 3))}
        return out


HEADS = [(256, 8, 2), (128, 16, 8), (64, 28, 4), (256, 3, 3)]
MIXES = {
    "one": ([1], [0]),
    "decode": ([1, 1, 1, 1, 1, 1], [0, 15, 16, 63, 64, 200]),
    "chunk": ([150], [37]),
    "prompts": ([64, 1, 0, 17, 128, 3, 1], [0, 5, 40, 127, 64, 250, 129]),
}


def run_prologue(ctx, rng, cache, batch, heads, n_dims, sections, positions=None, rows=None):
    d, kv, t = cache.head_dim, cache.kv_heads, batch.tokens
    x = rows or {"q_gate": rng.standard_normal((t, heads, 2, d)).astype(np.float32),
                 "key": rng.standard_normal((t, kv, d)).astype(np.float32),
                 "value": rng.standard_normal((t, kv, d)).astype(np.float32)}
    w = {n: (1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for n in ("q", "k")}
    pages, tables = DevicePages(ctx, cache), batch.device(ctx)
    blank = np.full((t, heads, d), -77.0, np.float32)
    q_out, g_out = ctx.buffer(blank), ctx.buffer(blank)
    bufs = [ctx.buffer(a) for a in (x["q_gate"], x["key"], x["value"], w["q"], w["k"])]
    pos = None if positions is None else ctx.buffer(positions.astype(np.int32))
    ctx.qwen35_attention_prologue_paged_q8_kv(
        *bufs, pos, pages.struct, tables, heads, n_dims, *sections, THETA, EPS, q_out, g_out)
    if positions is None:
        positions = np.zeros((4, t), np.int64)
        for _, first, count, length in po.live_sequences(cache, *batch.plain()):
            positions[:, first:first + count] = np.arange(length - count, length)
    q = po.norm_rope(x["q_gate"][:, :, 0], w["q"], positions, n_dims, sections, THETA, EPS)
    k = po.norm_rope(x["key"], w["k"], positions, n_dims, sections, THETA, EPS)
    exact = {"key": po.append(cache, "key", k, batch.plain()),
             "value": po.append(cache, "value", x["value"].astype(np.float64), batch.plain())}
    return (q, x["q_gate"][:, :, 1], q_out.download().reshape(blank.shape),
            g_out.download().reshape(blank.shape), pages, exact)


def check_pages(cache, got, exact):
    for name in ("key", "value"):
        want_s, got_s = cache.scales[name], got.scales[name]
        np.testing.assert_allclose(got_s, want_s, rtol=2.0 ** -19, atol=0)
        diff = got.codes[name].astype(np.int32) - cache.codes[name]
        for page, head, slot, dim in np.argwhere(diff != 0):
            slots, x = exact[name][page, head]  # a code that is not a new one must be equal
            value = x[slot - slots.start, dim]
            assert slots.start <= slot < slots.stop
            assert abs(diff[page, head, slot, dim]) == 1
            assert abs(value - np.floor(value) - 0.5) < 127 * 2.0 ** -18, (name, page, head, value)
        assert (diff != 0).mean() < 1e-3


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("d,heads,kv_heads", HEADS)
def test_prologue_into_pages(hip_ctx, d, heads, kv_heads, page_tokens, mix):
    rng = np.random.default_rng(d + heads + page_tokens)
    batch = Batch(rng, page_tokens, *MIXES[mix], gap=2)
    cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
    before = (cache.codes["key"].copy(), cache.codes["value"].copy())
    q, gate, got_q, got_g, pages, exact = run_prologue(hip_ctx, rng, cache, batch, heads, 64,
                                                       (11, 11, 10, 0))
    n = batch.rows
    size = np.abs(q[:n]).max(-1, keepdims=True)
    assert (np.abs(got_q[:n] - q[:n]) <= 2.0 ** -19 * size).all()
    np.testing.assert_array_equal(got_g[:n], gate[:n])
    assert (got_q[n:] == -77).all() and (got_g[n:] == -77).all()
    check_pages(cache, pages.read(), exact)
    del before


@pytest.mark.parametrize("page_tokens", [32, 128])
def test_prologue_positions_and_wide_rotation(hip_ctx, page_tokens):
    """Given MRoPE positions, far ones among them, and a rotation of the whole head."""
    rng = np.random.default_rng(9)
    batch = Batch(rng, page_tokens, [140, 5], [100, 0])
    for d, n_dims, sections in ((256, 256, (40, 40, 40, 8)), (128, 6, (1, 1, 1, 0)),
                                (64, 64, (11, 11, 10, 0))):
        cache = po.Pages(rng, batch.pages, page_tokens, 2, d)
        positions = rng.integers(0, 1 << 20, (4, batch.tokens))
        positions[:, -1] = (1 << 31) - 1
        q, _, got_q, _, pages, exact = run_prologue(hip_ctx, rng, cache, batch, 4, n_dims, sections,
                                                    positions=positions)
        size = np.abs(q).max(-1, keepdims=True)
        assert (np.abs(got_q - q) <= 2.0 ** -19 * size).all()
        check_pages(cache, pages.read(), exact)


def test_growing_scales_follow_the_plain_form(hip_ctx):
    """Token by token into one page, each 1.9 times the last: every step equals the
    plain form, and the page stays within a step of the rows."""
    rng = np.random.default_rng(10)
    cache = po.Pages(rng, 3, 16, 2, 64)
    pages = DevicePages(hip_ctx, cache)
    table = np.array([[1]], np.int32)
    rows = []
    for i in range(16):
        x = (rng.standard_normal((1, 2, 64)) * 1.9 ** i).astype(np.float32)
        rows.append(x[0])
        bufs = [hip_ctx.buffer(table), hip_ctx.buffer(np.array([0, 1], np.uint32)),
                hip_ctx.buffer(np.array([i + 1], np.uint32))]
        batch = kh.PagedBatch(*[b.view for b in bufs], 1, 1, 1, 1, 16)
        qg = rng.standard_normal((1, 2, 128)).astype(np.float32)
        w = np.ones(64, np.float32)
        out = [hip_ctx.buffer(byte_size=4 * 128) for _ in range(2)]
        hip_ctx.qwen35_attention_prologue_paged_q8_kv(
            hip_ctx.buffer(qg), hip_ctx.buffer(x), hip_ctx.buffer(x), hip_ctx.buffer(w),
            hip_ctx.buffer(w), None, pages.struct, batch, 2, 64, 11, 11, 10, 0, THETA, EPS, *out)
        po.append(cache, "value", x.astype(np.float64), (table, [0, 1], [i + 1], 1, 1, 16))
        got = pages.read()
        np.testing.assert_array_equal(got.scales["value"], cache.scales["value"])
        assert np.abs(got.codes["value"].astype(int) - cache.codes["value"]).max() <= 1
        cache.codes["value"] = got.codes["value"]  # ties may go either way once
        step = got.scales["value"][1].astype(np.float64)[:, None]
        assert (np.abs(got.values_of("value", 1)[:i + 1] - np.stack(rows)) <= step * 1.0001).all()


def test_prologue_values_out_of_the_ordinary(hip_ctx):
    """Zeros, tiny and huge rows, NaN and infinity, a NaN page that is begun again."""
    rng = np.random.default_rng(11)
    d, kv = 64, 2
    batch = Batch(rng, 16, [16, 16, 16, 16, 3, 1], [0, 0, 0, 0, 7, 16])
    cache = po.Pages(rng, batch.pages, 16, kv, d)
    cache.scales["value"][batch.table[0, 0]] = np.nan  # begun again below
    cache.scales["value"][batch.table[4, 0], 1] = 0.0  # older rows of zeros
    t = batch.tokens
    value = rng.standard_normal((t, kv, d)).astype(np.float32)
    value[16:32] = 0.0
    value[32:48] *= 1e-39
    value[48:64] *= 1e37
    value[64, 0, 5] = np.nan
    value[65, 0, 6] = np.inf
    rows = {"q_gate": rng.standard_normal((t, kv, 2, d)).astype(np.float32),
            "key": rng.standard_normal((t, kv, d)).astype(np.float32), "value": value}
    _, _, _, _, pages, exact = run_prologue(hip_ctx, rng, cache, batch, kv, 64, (11, 11, 10, 0),
                                            rows=rows)
    got = pages.read()
    check_pages(cache, got, exact)
    assert np.isnan(got.scales["value"][batch.table[4, 0], 0])
    assert (got.scales["value"][batch.table[2, 0]] == 0).all()
    assert np.isfinite(got.scales["value"][batch.table[0, 0]]).all()


def test_prologue_leaves_out_what_breaks_a_bound(hip_ctx):
    """Sequences past a bound and pages outside the pool: nothing of them changes."""
    rng = np.random.default_rng(12)
    for spoil in ("length", "query", "table", "width"):
        batch = Batch(rng, 16, [3, 20, 4], [10, 30, 13], gap=1)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        if spoil == "length":
            batch.max_keys = 40
        elif spoil == "query":
            batch.max_query = 8
        elif spoil == "table":
            batch.table[1, 2] = batch.pages
            batch.table[1, 3:] = -5
        else:
            batch.lengths[1] = 16 * batch.width + 1
            batch.max_keys = 1000
        q, _, got_q, _, pages, exact = run_prologue(hip_ctx, rng, cache, batch, 4, 64,
                                                    (11, 11, 10, 0))
        check_pages(cache, pages.read(), exact)
        written = np.zeros(batch.tokens, bool)
        for _, first, count, _ in po.live_sequences(cache, *batch.plain()):
            written[first:first + count] = True
        assert (got_q[~written] == -77).all() and (got_q[written] != -77).all()


# ------------------------------------------------------------- attention ----


def run_attention(ctx, cache, batch, heads, query, gate=None, f16=False):
    pages, tables = DevicePages(ctx, cache), batch.device(ctx)
    kind = np.float16 if f16 else np.float32
    out = ctx.buffer(np.full(query.shape, -77.0, kind))
    q = ctx.buffer(query)
    if f16:
        ctx.attention_f16q_paged_q8_kv(q, pages.struct, tables, heads, out)
    else:
        g = None if gate is None else ctx.buffer(gate)
        ctx.attention_f32_paged_q8_kv(q, g, pages.struct, tables, heads, out)
    return out.download(dtype=kind).reshape(query.shape).astype(np.float64)


def check_attention(ctx, rng, cache, batch, heads, f16, gated=False, spread=2.0):
    kind = np.float16 if f16 else np.float32
    query = (spread * rng.standard_normal((batch.tokens, heads, cache.head_dim))).astype(kind)
    gate = rng.standard_normal(query.shape).astype(np.float32) if gated else None
    got = run_attention(ctx, cache, batch, heads, query, gate, f16)
    want, size, score = po.attention(cache, query, batch.plain(), heads, gate)
    rows = ~np.isnan(size[..., 0])
    tol = po.attention_tolerance(size, want, score, cache.head_dim, f16)
    assert (got[~rows] == -77).all()
    off = np.abs(got - want)[rows] / tol[rows]
    assert (off <= 1).all(), (off.max(), np.argwhere(~(off <= 1))[:4])
    return got, want


ATTEND_MIXES = {
    "one": ([1], [0]),
    "decode": ([1, 1, 1, 1, 1, 1, 1], [0, 15, 16, 63, 64, 300, 1030]),
    "few": ([2, 4, 3], [0, 61, 777]),
    "chunk": ([150], [37]),
    "first": ([131], [0]),
    "prompts": ([64, 1, 0, 17, 130, 3, 1], [0, 5, 40, 127, 64, 250, 1500]),
}


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("mix", ATTEND_MIXES)
@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("d,heads,kv_heads", HEADS)
def test_attention_over_pages(hip_ctx, d, heads, kv_heads, page_tokens, mix, f16):
    rng = np.random.default_rng(d + heads + page_tokens)
    batch = Batch(rng, page_tokens, *ATTEND_MIXES[mix], gap=1)
    cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
    check_attention(hip_ctx, rng, cache, batch, heads, f16, gated=not f16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,heads,kv_heads,page_tokens", [(256, 16, 1, 32), (128, 5, 5, 128),
                                                         (64, 24, 2, 128), (128, 34, 2, 32)])
def test_attention_group_sizes(hip_ctx, d, heads, kv_heads, page_tokens, f16):
    rng = np.random.default_rng(d + heads)
    for new, before in (([1, 1], [400, 3]), ([9, 1, 70], [0, 333, 129])):
        batch = Batch(rng, page_tokens, new, before)
        cache = po.Pages(rng, batch.pages, page_tokens, kv_heads, d)
        check_attention(hip_ctx, rng, cache, batch, heads, f16)


@pytest.mark.parametrize("f16", [False, True])
def test_attention_peaked_and_far_apart_scales(hip_ctx, f16):
    """Scores of some hundreds (one key takes all), and value scales from 1e-20 to 1e3
    in neighbouring pages."""
    rng = np.random.default_rng(20)
    for new in ([1, 1, 1], [40, 1, 2]):
        batch = Batch(rng, 16, new, [500, 90, 33])
        cache = po.Pages(rng, batch.pages, 16, 2, 128)
        check_attention(hip_ctx, rng, cache, batch, 8, f16, spread=60.0)
        low, high = (-4, 1) if f16 else (-20, 3)
        cache.scales["value"] = (10.0 ** rng.uniform(low, high, cache.scales["value"].shape)).astype(
            np.float32)
        cache.scales["value"][batch.table[0, 3]] = 0.0
        cache.scales["key"][batch.table[0, 4]] = 0.0
        check_attention(hip_ctx, rng, cache, batch, 8, f16)


def test_attention_small_and_large_queries(hip_ctx):
    """Queries of 1e-30 and 1e+4 times the ordinary size: the parts that go into the
    matrix cores follow each row's magnitude."""
    rng = np.random.default_rng(21)
    for new in ([1, 1], [33, 1]):
        batch = Batch(rng, 64, new, [200, 70])
        cache = po.Pages(rng, batch.pages, 64, 2, 256)
        for spread in (0.0, 1e-30, 1e-3):
            check_attention(hip_ctx, rng, cache, batch, 8, False, spread=spread)
        cache.scales["key"] *= np.float32(1e-4)
        check_attention(hip_ctx, rng, cache, batch, 8, False, spread=1e4)


@pytest.mark.parametrize("f16", [False, True])
def test_attention_masked_places_hold_nothing(hip_ctx, f16):
    """NaN and infinite scales of pages behind the length, of spare pages, and codes of
    -128 behind a page's last token change nothing; pages outside the pool are not
    attended, and a sequence with no page inside gets zeros."""
    rng = np.random.default_rng(22)
    for new, before in (([1, 1, 1], [20, 39, 17]), ([30, 18, 12], [0, 22, 6])):
        batch = Batch(rng, 16, new, before, spare=3)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        used = set(batch.table[batch.table >= 0].tolist())
        for page in range(batch.pages):
            if page not in used:
                for n in ("key", "value"):
                    cache.scales[n][page] = (np.nan, np.inf)
        for b in range(len(new)):
            tail = int(batch.lengths[b]) % 16
            if tail:
                last = batch.table[b, (int(batch.lengths[b]) - 1) // 16]
                cache.codes["key"][last, :, tail:] = -128
                cache.codes["value"][last, :, tail:] = -128
        spare = [p for p in range(batch.pages) if p not in used][0]
        for b in range(len(new)):
            behind = -(-int(batch.lengths[b]) // 16)
            batch.table[b, behind:] = spare
        batch.table[1, 1] = batch.pages  # outside
        batch.table[2, :] = -1
        got, _ = check_attention(hip_ctx, rng, cache, batch, 4, f16)
        first = int(batch.starts[2])
        assert (got[first:first + new[2]] == 0).all()


def test_attention_nan_scale_reaches_its_rows_only(hip_ctx):
    rng = np.random.default_rng(23)
    batch = Batch(rng, 16, [1, 20, 1], [40, 30, 40])
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    cache.scales["value"][batch.table[1, 2], 1] = np.nan  # positions 32..47 of sequence 1
    query = rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)
    got = run_attention(hip_ctx, cache, batch, 4, query)
    bad = np.isnan(got).any(-1)
    want = np.zeros_like(bad)
    want[1 + 2:1 + 20, 2:] = True  # rows at positions 32 on, heads of KV head 1
    np.testing.assert_array_equal(bad, want)


def test_attention_leaves_out_what_breaks_a_bound(hip_ctx):
    rng = np.random.default_rng(24)
    for spoil in ("length", "query", "width", "starts"):
        batch = Batch(rng, 16, [3, 20, 4], [10, 30, 13], gap=1)
        cache = po.Pages(rng, batch.pages, 16, 2, 64)
        if spoil == "length":
            batch.max_keys = 40
        elif spoil == "query":
            batch.max_query = 8
        elif spoil == "width":
            batch.lengths[1] = 16 * batch.width + 1
            batch.max_keys = 1000
        else:
            batch.starts[3] = batch.tokens + 1
        check_attention(hip_ctx, rng, cache, batch, 4, False)


def test_shared_pages_and_long_sequences(hip_ctx):
    """A common prefix in shared pages, and one sequence of 9000 keys over few pages of
    the pool, each many times."""
    rng = np.random.default_rng(25)
    batch = Batch(rng, 64, [1, 1, 7], [130, 200, 128])
    batch.table[1, :2] = batch.table[0, :2]
    batch.table[2, :2] = batch.table[0, :2]
    cache = po.Pages(rng, batch.pages, 64, 2, 256)
    check_attention(hip_ctx, rng, cache, batch, 8, False)
    for new in ([1], [5], [40]):
        batch = Batch(rng, 64, new, [9000 - new[0]])
        batch.table[:] = rng.integers(0, 7, batch.table.shape)
        batch.pages = 7
        cache = po.Pages(rng, 7, 64, 1, 128)
        check_attention(hip_ctx, rng, cache, batch, 2, False)


def test_pool_beyond_32_bits(hip_ctx):
    """Pages whose bytes lie past 2^32 in a pool of 4.3 GiB a side."""
    torch = pytest.importorskip("torch")
    pages, pt, kv, d = 66000, 64, 4, 256
    keys = torch.zeros(pages, kv, pt, d, dtype=torch.int8, device="cuda")
    values = torch.zeros(pages, kv, pt // 8, d, 8, dtype=torch.int8, device="cuda")
    scales = [torch.full((pages, kv), 0.03, device="cuda") for _ in range(2)]
    rng = np.random.default_rng(26)
    batch = Batch(rng, pt, [1, 70], [130, 0])
    ids = np.array([65999, 3, 65998, 65997, 0], np.int32)
    batch.table = np.array([[65999, 3, 65998], [65997, 0, -1]], np.int32)
    cache = po.Pages(rng, 5, pt, kv, d)
    for i, page in enumerate(ids):
        keys[page] = torch.from_numpy(cache.codes["key"][i]).cuda()
        values[page] = torch.from_numpy(cache.device_values()[i]).cuda()
        for s, n in zip(scales, ("key", "value")):
            s[page] = torch.from_numpy(cache.scales[n][i]).cuda()
    torch.cuda.synchronize()
    struct = kh.PagedQ8Cache(*[kh.as_buffer(t) for t in (keys, values, *scales)], pages, pt, kv, d)
    query = rng.standard_normal((batch.tokens, 8, d)).astype(np.float32)
    out = hip_ctx.buffer(byte_size=query.nbytes)
    tables = batch.device(hip_ctx)
    hip_ctx.attention_f32_paged_q8_kv(hip_ctx.buffer(query), None, struct, tables, 8, out)
    batch.table = np.array([[0, 1, 2], [3, 4, -1]], np.int32)
    want, size, score = po.attention(cache, query, batch.plain(), 8)
    tol = po.attention_tolerance(size, want, score, d, False)
    assert (np.abs(out.download().reshape(query.shape) - want) <= tol).all()
    rows = [hip_ctx.buffer(byte_size=2 * 5 * pt * kv * d) for _ in range(2)]
    hip_ctx.dequantize_kv_pages_q8_f16(struct, hip_ctx.buffer(ids), 5, *rows)
    for r, n in zip(rows, ("key", "value")):
        got = r.download(dtype=np.float16).reshape(5, pt, kv, d)
        for i in range(5):
            np.testing.assert_array_equal(got[i], cache.values_of(n, i).astype(np.float32).astype(
                np.float16))


@pytest.mark.parametrize("d,page_tokens", [(64, 16), (128, 32), (256, 128)])
def test_pages_read_back(hip_ctx, d, page_tokens):
    """Exact: a code times a scale in f32, rounded once more to f16.  The 64-bit product
    rounded to f32 is the f32 product."""
    rng = np.random.default_rng(d)
    cache = po.Pages(rng, 6, page_tokens, 3, d)
    cache.scales["key"][4, 1] = np.nan
    pages = DevicePages(hip_ctx, cache)
    ids = np.array([4, 0, 6, 4, -1, 5], np.int32)
    out = [hip_ctx.buffer(np.full(6 * page_tokens * 3 * d, 9, np.float16)) for _ in range(2)]
    hip_ctx.dequantize_kv_pages_q8_f16(pages.struct, hip_ctx.buffer(ids), 6, *out)
    for o, n in zip(out, ("key", "value")):
        got = o.download(dtype=np.float16).reshape(6, page_tokens, 3, d)
        for i, page in enumerate(ids):
            want = (cache.values_of(n, page) if po.inside(cache, page)
                    else np.zeros((page_tokens, 3, d)))
            np.testing.assert_array_equal(got[i], want.astype(np.float32).astype(np.float16))


# ---------------------------------------------------------- used together ----


def test_prompt_then_decode_steps(hip_ctx):
    """A prompt in ragged chunks, then single tokens of three sequences, appended and
    attended as a server does: each step's attention equals the plain form over the
    pages that the device holds, and those are within a step of the rows."""
    rng = np.random.default_rng(30)
    d, heads, kv, pt, longest = 128, 8, 2, 16, 112
    cache = po.Pages(rng, 3 * 7 + 2, pt, kv, d)
    pages = DevicePages(hip_ctx, cache)
    table = rng.permutation(cache.pages)[:21].reshape(3, 7).astype(np.int32)
    w = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    have = [0, 0, 0]
    rows = [[], [], []]
    for new in ([30, 1, 0], [33, 17, 50], [1, 1, 1], [1, 0, 1], [1, 1, 1], [3, 40, 1], [1, 1, 1]):
        batch = Batch(rng, pt, new, have)
        batch.table, batch.width, batch.pages = table, 7, cache.pages
        batch.max_keys = longest
        t = batch.tokens
        x = {"qg": rng.standard_normal((t, heads, 2 * d)).astype(np.float32),
             "k": rng.standard_normal((t, kv, d)).astype(np.float32),
             "v": rng.standard_normal((t, kv, d)).astype(np.float32)}
        tables = batch.device(hip_ctx)
        q, g, out = (hip_ctx.buffer(byte_size=4 * t * heads * d) for _ in range(3))
        bufs = [hip_ctx.buffer(a) for a in (x["qg"], x["k"], x["v"], w, w)]
        hip_ctx.begin_graph()
        hip_ctx.qwen35_attention_prologue_paged_q8_kv(*bufs, None, pages.struct, tables, heads, 64,
                                                      11, 11, 10, 0, THETA, EPS, q, g)
        hip_ctx.attention_f32_paged_q8_kv(q, g, pages.struct, tables, heads, out)
        hip_ctx.commit_graph()
        held = pages.read()
        shape = (t, heads, d)
        query, gate = q.download().reshape(shape), g.download().reshape(shape)
        want, size, score = po.attention(held, query, batch.plain(), heads, gate)
        tol = po.attention_tolerance(size, want, score, d, False)
        assert (np.abs(out.download().reshape(shape) - want) <= tol).all()
        for b in range(3):
            rows[b] += list(x["v"][batch.starts[b]:batch.starts[b + 1]])
            have[b] += new[b]
            for p in range(-(-have[b] // pt)):
                got = held.values_of("value", table[b, p])[:have[b] - p * pt]
                step = held.scales["value"][table[b, p]].astype(np.float64)[:, None]
                assert (np.abs(got - np.stack(rows[b][p * pt:(p + 1) * pt])) <= step).all()


def test_captured_step_replays_with_new_arrays(hip_ctx):
    """Append and attention captured once; replays with other rows, lengths and tables
    in the same buffers equal the eager calls, with eager work between them."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(31)
    d, heads, kv, pt = 128, 8, 2, 16
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    lengths = [[40, 300, 17], [41, 301, 18], [60, 160, 250], [1, 2, 320]]
    cache = po.Pages(rng, 64, pt, kv, d)
    w = torch.ones(d, device="cuda")
    t = 3

    def arrays(seed, step):
        r = np.random.default_rng(seed)
        return {"qg": r.standard_normal((t, heads, 2 * d)).astype(np.float32),
                "k": r.standard_normal((t, kv, d)).astype(np.float32),
                "v": r.standard_normal((t, kv, d)).astype(np.float32),
                "table": r.permutation(64)[:60].reshape(3, 20).astype(np.int32),
                "starts": np.arange(4, dtype=np.int32),
                "lengths": np.array(lengths[step], np.int32)}

    def device():
        s = {k: torch.from_numpy(v).cuda() for k, v in arrays(0, 0).items()}
        s.update(keys=torch.from_numpy(cache.codes["key"]).cuda(),
                 values=torch.from_numpy(cache.device_values()).cuda(),
                 ks=torch.from_numpy(cache.scales["key"]).cuda(),
                 vs=torch.from_numpy(cache.scales["value"]).cuda())
        for n in ("q", "g", "out"):
            s[n] = torch.empty(t, heads, d, device="cuda")
        return s

    def step(s):
        c = kh.PagedQ8Cache(*[kh.as_buffer(s[n]) for n in ("keys", "values", "ks", "vs")], 64, pt,
                            kv, d)
        b = kh.PagedBatch(*[kh.as_buffer(s[n]) for n in ("table", "starts", "lengths")], 3, 20, t,
                          1, 320)
        ctx.qwen35_attention_prologue_paged_q8_kv(s["qg"], s["k"], s["v"], w, w, None, c, b, heads,
                                                  64, 11, 11, 10, 0, THETA, EPS, s["q"], s["g"])
        ctx.attention_f32_paged_q8_kv(s["q"], s["g"], c, b, heads, s["out"])

    eager, captured = device(), device()
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(captured)
        for i in range(len(lengths)):
            for k, v in arrays(50 + i, i).items():
                eager[k].copy_(torch.from_numpy(v))
                captured[k].copy_(torch.from_numpy(v))
            graph.replay()
            step(eager)
            stream.synchronize()
            for k in ("keys", "values", "ks", "vs", "q", "g", "out"):
                assert torch.equal(eager[k], captured[k]), (i, k)
    ctx.commit_graph()
    ctx.close()
