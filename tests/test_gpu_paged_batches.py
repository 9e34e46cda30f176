"""Batches over the paged 8-bit KV cache that the other tests leave out: appends of more
sequences than a wave looks through at a time, into pages beyond 2^32 bytes, pages that a
batch does not touch, and sampled rows beyond 2^32 bytes.  Tolerances are those of
tests/test_gpu_paged_q8.py and tests/test_gpu_sample.py."""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
from test_gpu_paged_q8 import (EPS, THETA, Batch, DevicePages, check_attention, check_pages,
                                run_prologue)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences", [64, 65, 200])
def test_appends_of_many_sequences(hip_ctx, sequences):
    """Single tokens, chunks and sequences without any, and pages that none of them
    appends to, which keep every byte."""
    rng = np.random.default_rng(sequences)
    new = rng.integers(0, 9, sequences)
    new[::3] = 1
    new[-1] = 40
    before = rng.integers(0, 100, sequences)
    batch = Batch(rng, 16, new.tolist(), before.tolist(), spare=5, gap=3)
    cache = po.Pages(rng, batch.pages, 16, 2, 64)
    held = ({n: c.copy() for n, c in cache.codes.items()},
            {n: s.copy() for n, s in cache.scales.items()})
    q, gate, got_q, got_g, pages, exact = run_prologue(hip_ctx, rng, cache, batch, 4, 64,
                                                       (11, 11, 10, 0))
    got, n = pages.read(), batch.rows
    check_pages(cache, got, exact)
    assert (np.abs(got_q[:n] - q[:n]) <= 2.0 ** -19 * np.abs(q[:n]).max(-1, keepdims=True)).all()
    np.testing.assert_array_equal(got_g[:n], gate[:n])
    assert (got_q[n:] == -77).all() and (got_g[n:] == -77).all()
    touched = {int(batch.table[b, p]) for b in range(sequences) if new[b]
               for p in range(before[b] // 16, (before[b] + new[b] - 1) // 16 + 1)}
    rest = [p for p in range(batch.pages) if p not in touched]
    assert len(rest) > 5
    for name in ("key", "value"):
        np.testing.assert_array_equal(got.codes[name][rest], held[0][name][rest])
        np.testing.assert_array_equal(got.scales[name][rest], held[1][name][rest])


@pytest.mark.parametrize("group", [7, 150])
def test_attention_of_many_sequences_and_heads(hip_ctx, group):
    """200 sequences; 150 query heads of a KV head are more than a tile's rows for each
    token."""
    rng = np.random.default_rng(group)
    new = rng.integers(0, 3, 200)
    before = rng.integers(0, 120, 200)
    new[5], before[5] = 30, 700
    batch = Batch(rng, 32, new.tolist(), before.tolist(), gap=1)
    cache = po.Pages(rng, batch.pages, 32, 1, 64)
    check_attention(hip_ctx, rng, cache, batch, group, group == 7, gated=group != 7)


def test_appends_beyond_32_bits(hip_ctx):
    """A chunk and a token into pages whose bytes lie past 2^32 in a pool of 4.3 GiB a
    side, equal to the same rows in a small pool."""
    torch = pytest.importorskip("torch")
    pages, pt, kv, d, heads = 66000, 64, 4, 256, 4
    rng = np.random.default_rng(81)
    batch = Batch(rng, pt, [1, 70], [130, 40])
    small = po.Pages(rng, 5, pt, kv, d)
    ids = np.array([65999, 3, 65998, 65997, 2], np.int64)
    t = batch.tokens
    rows = [rng.standard_normal(s).astype(np.float32)
            for s in ((t, heads, 2 * d), (t, kv, d), (t, kv, d))]
    w = np.ones(d, np.float32)
    got = []
    for count, place in ((5, np.arange(5)), (pages, ids)):
        keys = torch.zeros(count, kv, pt, d, dtype=torch.int8, device="cuda")
        values = torch.zeros(count, kv, pt // 8, d, 8, dtype=torch.int8, device="cuda")
        scales = [torch.full((count, kv), 0.03, device="cuda") for _ in range(2)]
        for i, page in enumerate(place):
            keys[page] = torch.from_numpy(small.codes["key"][i]).cuda()
            values[page] = torch.from_numpy(small.device_values()[i]).cuda()
            for s, n in zip(scales, ("key", "value")):
                s[page] = torch.from_numpy(small.scales[n][i]).cuda()
        batch.table = np.array([[place[0], place[1], place[2]], [place[3], place[4], -1]], np.int32)
        struct = kh.PagedQ8Cache(*[kh.as_buffer(x) for x in (keys, values, *scales)], count, pt, kv,
                                 d)
        out = [torch.zeros(t, heads, d, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        hip_ctx.qwen35_attention_prologue_paged_q8_kv(
            *[hip_ctx.buffer(x) for x in (*rows, w, w)], None, struct, batch.device(hip_ctx), heads,
            64, 11, 11, 10, 0, THETA, EPS, *out)
        torch.cuda.synchronize()
        place = torch.from_numpy(place).cuda()
        got.append([x[place].cpu() for x in (keys, values, *scales)] + [x.cpu() for x in out])
        del keys, values
    for x, y in zip(*got):
        assert torch.equal(x, y)
    assert not np.array_equal(got[0][0].numpy(), small.codes["key"])


def test_sampled_rows_beyond_32_bits(hip_ctx):
    """Three rows 2^31 floats apart draw as they do side by side."""
    torch = pytest.importorskip("torch")
    size, stride = 5000, 2 ** 31
    rng = np.random.default_rng(82)
    x = torch.from_numpy((2 * rng.standard_normal((3, size))).astype(np.float32)).cuda()
    far = torch.empty(2 * stride + size, device="cuda")
    for r in range(3):
        far[r * stride:r * stride + size] = x[r]
    u = torch.from_numpy(rng.random(3).astype(np.float32)).cuda()
    p = torch.tensor([0.9, 1.0, 0.5], device="cuda")
    got = []
    torch.cuda.synchronize()
    for logits, step in ((x, size), (far, stride)):
        token = torch.full((3,), -7, device="cuda", dtype=torch.int32)
        share = torch.full((3,), -7.0, device="cuda")
        torch.cuda.synchronize()
        hip_ctx.sample_f32_i32(logits, 3, size, step, None, None, p, None, u, token, share)
        torch.cuda.synchronize()
        got.append((token, share))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert (got[0][0] >= 0).all()


def test_the_most_rows(hip_ctx):
    """67108864 query rows, the most that the attention takes: two tokens of 1024 heads and
    65534 rows of no sequence, in a batch that has its results joined.  The rows of no
    sequence stay as they were."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(83)
    heads, d, pt, kv = 1024, 64, 16, 256
    tokens = 65536
    batch = Batch(rng, pt, [1, 1], [200, 299])
    cache = po.Pages(rng, batch.pages, pt, kv, d)
    query = torch.zeros(tokens, heads, d, device="cuda", dtype=torch.float16)
    query[:2] = torch.from_numpy(rng.standard_normal((2, heads, d)).astype(np.float16)).cuda()
    out = torch.full((tokens, heads, d), -77.0, device="cuda", dtype=torch.float16)
    batch.tokens = tokens
    pages, tables = DevicePages(hip_ctx, cache), batch.device(hip_ctx)
    torch.cuda.synchronize()
    hip_ctx.attention_f16q_paged_q8_kv(query, pages.struct, tables, heads, out)
    torch.cuda.synchronize()
    got, held = out[:2].cpu().numpy().astype(np.float64), query[:2].cpu().numpy()
    assert bool((out[2:] == -77).all())
    batch.tokens = 2
    want, size, score = po.attention(cache, held, batch.plain(), heads)
    tol = po.attention_tolerance(size, want, score, d, True)
    assert (np.abs(got - want) <= tol).all()
