"""Argument checks of the entries for shared prefixes, key weights, eviction and log
probabilities (no GPU), and closed forms of the plain implementations that the GPU tests
compare with."""
import math

import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so
from test_paged_cpu import (ACCEPTED, BATCH_ERRORS, CACHE_ERRORS, attend, batch_of, cache_of, fake)

NO = kh.KrakenBuffer(None, 0)


@pytest.fixture()
def vctx():
    ctx = kh.Context(validation_only=True)
    yield ctx
    ctx.close()


def prefixes_of(groups=2, max_rows=7, max_prefix=64, **over):
    b = dict(starts=fake(4 * (groups + 1)), lengths=fake(4 * groups))
    b.update(over)
    return kh.SharedPrefixes(b["starts"], b["lengths"], groups, max_rows, max_prefix)


def shared(f16=False, prefixes=None, **kw):
    args = list(attend(f16=f16, **kw))
    args.insert(4 - f16, prefixes or prefixes_of())
    return args


def weigh(f16=False, window=0, decay=1.0, stride=128, cache=None, batch=None, heads=8, **over):
    b = dict(q=fake((2 if f16 else 4) * 7 * 8 * 256), w=fake(4 * 3 * 2 * stride))
    b.update(over)
    return (b["q"], cache or cache_of(), batch or batch_of(), heads, window, decay, b["w"], stride)


def select(**over):
    a = dict(weights=fake(4 * 3 * 2 * 90), weight_stride=90, lengths=fake(12), keep=fake(12),
             sequences=3, kv_heads=2, max_keys=80, first=4, last=5, kept=fake(4 * 3 * 2 * 40, 0x100000),
             kept_stride=40, kept_lengths=fake(12, 0x200000))
    a.update(over)
    return list(a.values())


def gather(**over):
    a = dict(cache=cache_of(), table=fake(4 * 3 * 2), width=2, kept=fake(4 * 3 * 2 * 40),
             kept_lengths=fake(12), kept_stride=40, sequences=3, target=fake(12), target_width=1,
             weights=fake(4 * 3 * 2 * 90), stride=90, output=fake(4 * 3 * 2 * 90, 0x100000))
    a.update(over)
    return list(a.values())


def score(**over):
    a = dict(logits=fake(4 * 25), rows=3, size=5, stride=10, temperature=fake(12),
             tokens=fake(12), top=4, logprob=fake(12, 0x100000), rank=fake(12, 0x200000),
             entropy=fake(12, 0x300000), top_tokens=fake(48, 0x400000),
             top_logprobs=fake(48, 0x500000))
    a.update(over)
    return list(a.values())


def refused(vctx, name, args, fragment):
    assert vctx.status(name, *args) == kh.INVALID_ARGUMENT, name
    assert fragment in kh.last_error(), (name, kh.last_error())


@pytest.mark.parametrize("kw,fragment", CACHE_ERRORS)
def test_cache_refusals(vctx, kw, fragment):
    c = cache_of(**kw)
    for name, args in (("attention_f32_shared_paged_q8_kv", shared(cache=c)),
                       ("attention_f16q_shared_paged_q8_kv", shared(True, cache=c)),
                       ("key_weights_f32_paged_q8_kv", weigh(cache=c)),
                       ("key_weights_f16q_paged_q8_kv", weigh(True, cache=c)),
                       ("gather_kv_pages_q8", gather(cache=c))):
        refused(vctx, name, args, fragment)


@pytest.mark.parametrize("kw,fragment", BATCH_ERRORS)
def test_batch_refusals(vctx, kw, fragment):
    b = batch_of(**kw)
    for name, args in (("attention_f32_shared_paged_q8_kv", shared(batch=b)),
                       ("attention_f16q_shared_paged_q8_kv", shared(True, batch=b)),
                       ("key_weights_f32_paged_q8_kv", weigh(batch=b)),
                       ("key_weights_f16q_paged_q8_kv", weigh(True, batch=b))):
        refused(vctx, name, args, fragment)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("kw,fragment", [
    (dict(heads=0), "dimensions must be positive"),
    (dict(heads=5), "divisible by kv_heads"),
    (dict(q=fake(64)), "query buffer is too small"),
    (dict(o=NO), "output buffer is not initialized"),
    (dict(q=fake(1 << 20, 0x1004)), "buffers must be 16-byte aligned"),
    (dict(batch=batch_of(tokens=(1 << 17) + 1), o=fake(1 << 62), q=fake(1 << 62)),
     "takes up to 1048576 query rows"),
    (dict(prefixes=prefixes_of(groups=0)), "prefix dimensions must be positive"),
    (dict(prefixes=prefixes_of(max_rows=0)), "prefix dimensions must be positive"),
    (dict(prefixes=prefixes_of(max_prefix=0)), "prefix dimensions must be positive"),
    (dict(prefixes=prefixes_of(groups=4)), "no more groups than sequences"),
    (dict(prefixes=prefixes_of(starts=fake(11))), "group starts buffer is too small"),
    (dict(prefixes=prefixes_of(lengths=NO)), "prefix lengths buffer is not initialized"),
])
def test_shared_attention_refusals(vctx, kw, fragment, f16):
    name = "attention_f16q_shared_paged_q8_kv" if f16 else "attention_f32_shared_paged_q8_kv"
    refused(vctx, name, shared(f16, **kw), fragment)


def test_shared_attention_null_structs(vctx):
    for at, fragment in ((2, "cache must not be null"), (3, "batch must not be null")):
        args = shared()
        args[at] = None
        refused(vctx, "attention_f32_shared_paged_q8_kv", args, fragment)
    q, g, cache, batch, heads, o = attend()
    refused(vctx, "attention_f32_shared_paged_q8_kv", (q, g, cache, batch, None, heads, o),
            "prefixes must not be null")
    refused(vctx, "attention_f32_shared_paged_q8_kv",
            (q, fake(8), cache, batch, prefixes_of(), heads, o), "gate buffer is too small")


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("kw,fragment", [
    (dict(heads=0), "dimensions must be positive"),
    (dict(heads=3), "divisible by kv_heads"),
    (dict(q=fake(64)), "query buffer is too small"),
    (dict(q=fake(1 << 20, 0x1008)), "buffers must be 16-byte aligned"),
    (dict(decay=-0.5), "decay must be finite and not negative"),
    (dict(decay=math.inf), "decay must be finite and not negative"),
    (dict(decay=math.nan), "decay must be finite and not negative"),
    (dict(stride=0), "stride must be positive"),
    (dict(stride=1 << 62), "value count overflow"),
    (dict(w=fake(4 * 3 * 2 * 128 - 4)), "output buffer is too small"),
    (dict(w=NO), "output buffer is not initialized"),
])
def test_key_weight_refusals(vctx, kw, fragment, f16):
    name = "key_weights_f16q_paged_q8_kv" if f16 else "key_weights_f32_paged_q8_kv"
    refused(vctx, name, weigh(f16, **kw), fragment)


@pytest.mark.parametrize("kw,fragment", [
    (dict(sequences=0), "dimensions must be positive"),
    (dict(kv_heads=0), "dimensions must be positive"),
    (dict(max_keys=0), "dimensions must be positive"),
    (dict(kept_stride=0), "dimensions must be positive"),
    (dict(max_keys=1 << 31), "keys exceed int32 range"),
    (dict(sequences=(1 << 19) + 1), "takes up to 1048576 pairs"),
    (dict(kv_heads=1 << 40), "takes up to 1048576 pairs"),
    (dict(weight_stride=79), "weight stride must be at least max_keys"),
    (dict(weight_stride=1 << 62), "value count overflow"),
    (dict(kept_stride=1 << 62), "value count overflow"),
    (dict(weights=fake(64)), "weights buffer is too small"),
    (dict(lengths=fake(8)), "lengths buffer is too small"),
    (dict(keep=NO), "keep buffer is not initialized"),
    (dict(kept=fake(4 * 3 * 2 * 40 - 4)), "output buffer is too small"),
    (dict(kept_lengths=fake(8)), "output lengths buffer is too small"),
    (dict(kept_lengths=fake(12)), "must not overlap"),  # the lengths in place
    (dict(keep=fake(12, 0x200008)), "must not overlap"),
    (dict(kept=fake(4 * 3 * 2 * 40, 0x1000 + 4 * 3 * 2 * 90 - 4)), "must not overlap"),
    (dict(kept=fake(4 * 3 * 2 * 40, 0x200000 - 4 * 3 * 2 * 40 + 4)), "must not overlap"),
])
def test_select_refusals(vctx, kw, fragment):
    refused(vctx, "select_keys_f32_i32", select(**kw), fragment)


@pytest.mark.parametrize("kw,fragment", [
    (dict(width=0), "dimensions must be positive"),
    (dict(kept_stride=0), "dimensions must be positive"),
    (dict(sequences=0), "dimensions must be positive"),
    (dict(target_width=0), "dimensions must be positive"),
    (dict(sequences=(1 << 19) + 1), "takes up to 1048576 pairs"),
    (dict(target_width=1 << 31), "table width exceeds int32 range"),
    (dict(kept_stride=1 << 62), "value count overflow"),
    (dict(table=fake(20)), "page table buffer is too small"),
    (dict(kept=fake(4 * 3 * 2 * 40 - 1)), "positions buffer is too small"),
    (dict(kept_lengths=NO), "lengths buffer is not initialized"),
    (dict(target=fake(8)), "target table buffer is too small"),
    (dict(weights=NO), "takes weights and their output together"),
    (dict(output=NO), "takes weights and their output together"),
    (dict(stride=0), "weight stride must be positive"),
    (dict(stride=1 << 62), "value count overflow"),
    (dict(weights=fake(64)), "weights buffer is too small"),
    (dict(output=fake(64, 0x100000)), "weights output buffer is too small"),
    (dict(output=fake(4 * 3 * 2 * 90)), "must not overlap"),
    (dict(output=fake(4 * 3 * 2 * 90, 0x1000 + 4 * 3 * 2 * 90 - 4)), "must not overlap"),
    (dict(kept=fake(4 * 3 * 2 * 40, 0x100000)), "must not overlap"),
    (dict(target=fake(12, 0x100000 + 4 * 3 * 2 * 90 - 4)), "must not overlap"),
])
def test_gather_refusals(vctx, kw, fragment):
    refused(vctx, "gather_kv_pages_q8", gather(**kw), fragment)


@pytest.mark.parametrize("kw,fragment", [
    (dict(rows=0), "dimensions must be positive"),
    (dict(size=0), "dimensions must be positive"),
    (dict(stride=4), "row stride must be at least the row size"),
    (dict(stride=1 << 63), "value count overflow"),
    (dict(logits=fake(1 << 40), rows=1, size=(1 << 22) + 1, stride=1 << 23),
     "rows of up to 4194304 logits"),
    (dict(logits=fake(1 << 40), rows=65536), "rows of up to 4194304 logits"),
    (dict(top=33), "lists up to 32 tokens"),
    (dict(logits=fake(96)), "logits buffer is too small"),
    (dict(logprob=NO, rank=NO, entropy=NO, top_tokens=NO, top_logprobs=NO), "has no output"),
    (dict(tokens=NO), "takes tokens exactly with their outputs"),
    (dict(logprob=NO, rank=NO), "takes tokens exactly with their outputs"),
    (dict(top=0), "number of top tokens exactly with their outputs"),
    (dict(top_tokens=NO, top_logprobs=NO), "number of top tokens exactly with their outputs"),
    (dict(temperature=fake(8)), "temperature buffer is too small"),
    (dict(tokens=fake(8)), "tokens buffer is too small"),
    (dict(logprob=fake(8)), "logprob output buffer is too small"),
    (dict(rank=fake(8)), "rank output buffer is too small"),
    (dict(entropy=fake(8)), "entropy output buffer is too small"),
    (dict(top_tokens=fake(44)), "top token output buffer is too small"),
    (dict(top_logprobs=fake(44, 0x500000)), "top logprob output buffer is too small"),
    (dict(rank=fake(12)), "must not overlap"),  # the tokens in place
    (dict(entropy=fake(12, 0x1000 + 4 * 25 - 4)), "must not overlap"),
    (dict(temperature=fake(12, 0x100008)), "must not overlap"),
    (dict(rank=fake(12, 0x400000 + 44)), "must not overlap"),
    (dict(top_logprobs=fake(48, 0x400000)), "must not overlap"),
])
def test_logprob_refusals(vctx, kw, fragment):
    refused(vctx, "token_logprobs_f32", score(**kw), fragment)


def test_accepted(vctx):
    for name, args in (
            ("attention_f32_shared_paged_q8_kv", shared()),
            ("attention_f32_shared_paged_q8_kv", shared(g=NO)),
            ("attention_f16q_shared_paged_q8_kv", shared(True)),
            ("key_weights_f32_paged_q8_kv", weigh(window=1 << 40)),
            ("key_weights_f16q_paged_q8_kv", weigh(True, decay=0.0)),
            ("select_keys_f32_i32", select()),
            ("select_keys_f32_i32", select(first=1 << 40, last=1 << 40)),
            ("gather_kv_pages_q8", gather()),
            ("gather_kv_pages_q8", gather(weights=NO, output=NO, stride=0)),
            ("token_logprobs_f32", score()),
            ("token_logprobs_f32", score(temperature=NO, top_tokens=NO)),
            ("token_logprobs_f32", score(tokens=NO, logprob=NO, rank=NO)),
            ("token_logprobs_f32", score(top=0, top_tokens=NO, top_logprobs=NO))):
        assert vctx.status(name, *args) == kh.UNAVAILABLE, (name, kh.last_error())
        assert kh.last_error() == ACCEPTED


# ------------------------------------------------------- the plain forms ----


def test_plain_key_weights_closed_forms():
    """A zero query weighs its keys alike; each row's weights sum to one."""
    rng = np.random.default_rng(1)
    cache = po.Pages(rng, 3, 16, 2, 64)
    batch = (np.array([[2, 0]], np.int32), [0, 3], [19], 3, 3, 32)
    old = rng.random((1, 2, 32)).astype(np.float32)
    got, _ = so.key_weights(cache, np.zeros((3, 4, 64)), batch, 4, 0, 0.5, old, 32)
    want = np.array([sum(2 / (17 + i) for i in range(3) if j <= 16 + i) for j in range(19)])
    want = want + np.where(np.arange(19) < 16, 0.5 * old[..., :19].astype(np.float64), 0)
    np.testing.assert_allclose(got[..., :19], want, rtol=1e-12)
    np.testing.assert_array_equal(got[..., 19:], old[..., 19:])
    got, _ = so.key_weights(cache, rng.standard_normal((3, 4, 64)), batch, 4, 2, 0.0, old, 32)
    np.testing.assert_allclose(got[..., :19].sum(-1), 4.0)  # two rows, two heads


def test_plain_selection_known_answers():
    w = np.array([[[5, 1, 9, 2, 2, 7, 2, 3]]], np.float32)
    for keep, first, last, want in ((4, 1, 1, [0, 2, 5, 7]), (5, 0, 0, [0, 2, 3, 5, 7]),
                                    (3, 2, 2, [0, 6, 7]), (1, 5, 3, [7]), (0, 1, 1, []),
                                    (8, 0, 0, list(range(8))), (5, 0, 1, [0, 2, 3, 5, 7])):
        kept, n = so.select_keys(w, [8], [keep], 8, first, last, 8)
        assert n[0] == keep and kept[0, 0, :keep].tolist() == want
    w[0, 0, 2] = np.nan
    kept, _ = so.select_keys(w, [8], [7], 8, 0, 0, 8)
    assert 2 not in kept[0, 0, :7]


def test_plain_gather_moves_no_value_by_more_than_half_a_step():
    rng = np.random.default_rng(2)
    cache = po.Pages(rng, 6, 16, 2, 64)
    before = {n: np.concatenate([cache.values_of(n, p) for p in (4, 1, 0)]) for n in ("key", "value")}
    kept = np.stack([np.sort(rng.permutation(48)[:21]) for _ in range(2)])[None].astype(np.int32)
    so.gather(cache, np.array([[4, 1, 0]]), kept, [21], 21, np.array([[5, 2]]))
    for n in ("key", "value"):
        got = np.concatenate([cache.values_of(n, p) for p in (5, 2)])
        for h in range(2):
            step = np.repeat(cache.scales[n][[5, 2], h], 16)[:21, None].astype(np.float64)
            assert (np.abs(got[:21, h] - before[n][kept[0, h], h]) <= 0.5 * step * 1.00001).all()
            assert (got[21:, h] == 0).all()
            assert cache.scales[n][5, h] in cache.scales[n][[4, 1, 0], h]


def test_plain_logprobs_known_answers():
    x = np.log([0.1, 0.4, 0.2, 0.3])
    got = so.logprobs(x, 1.0, 2, 3)
    assert got["rank"] == 2 and got["top_tokens"] == [1, 3, 2]
    np.testing.assert_allclose(got["logprob"], math.log(0.2))
    np.testing.assert_allclose(got["entropy"], -sum(p * math.log(p) for p in (.1, .4, .2, .3)))
    np.testing.assert_allclose(got["top_logprobs"], np.log([0.4, 0.3, 0.2]))
    got = so.logprobs([1.0, math.nan, math.inf, math.inf, -math.inf], 0.5, 1, 5)
    assert got["rank"] == 4 and got["logprob"] == -math.inf
    assert got["top_tokens"] == [2, 3, 0, 4, 5]
    np.testing.assert_allclose(got["top_logprobs"][:2], [math.log(0.5)] * 2)
    np.testing.assert_allclose(got["entropy"], math.log(2))
    assert so.logprobs([math.nan] * 3, 1.0, 0, 1)["top_tokens"] == [3]


def test_plain_shared_tables_begin_alike():
    from test_gpu_paged_q8 import Batch
    rng = np.random.default_rng(3)
    batch = Batch(rng, 16, [0, 1, 2, 1], [64, 50, 48, 3])
    starts, lengths = so.share_prefixes(16, batch, [(0, 3, 55)])
    assert starts.tolist() == [0, 3] and lengths.tolist() == [55]
    assert (batch.table[0, :3] == batch.table[1, :3]).all()
    assert (batch.table[2, :3] == batch.table[1, :3]).all()
    assert (batch.table[0, 3] != batch.table[1, 3])
