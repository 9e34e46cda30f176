"""Argument checks of the paged 8-bit cache's entries and of sampling (no GPU), and
closed forms of the plain implementations that the GPU tests compare with."""
import math

import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po

ACCEPTED = "validation-only context: arguments accepted"


@pytest.fixture()
def vctx():
    ctx = kh.Context(validation_only=True)
    yield ctx
    ctx.close()


def fake(nbytes, at=0x1000):
    return kh.KrakenBuffer(at, nbytes)


def cache_of(pages=5, pt=64, kv=2, d=256, **over):
    b = dict(kp=fake(pages * pt * kv * d), vp=fake(pages * pt * kv * d), ks=fake(4 * pages * kv),
             vs=fake(4 * pages * kv))
    b.update(over)
    return kh.PagedQ8Cache(b["kp"], b["vp"], b["ks"], b["vs"], pages, pt, kv, d)


def batch_of(sequences=3, width=2, tokens=7, max_query=4, max_keys=128, **over):
    b = dict(table=fake(4 * sequences * width), starts=fake(4 * (sequences + 1)),
             lengths=fake(4 * sequences))
    b.update(over)
    return kh.PagedBatch(b["table"], b["starts"], b["lengths"], sequences, width, tokens,
                         max_query, max_keys)


def prologue(cache=None, batch=None, heads=8, n_dims=64, sections=(11, 11, 10, 0), theta=1e7,
             tokens=7, d=256, kv=2, **over):
    b = dict(qg=fake(8 * tokens * heads * d), k=fake(4 * tokens * kv * d),
             v=fake(4 * tokens * kv * d), qn=fake(4 * d), kn=fake(4 * d), pos=fake(16 * tokens),
             qo=fake(4 * tokens * heads * d), go=fake(4 * tokens * heads * d))
    b.update(over)
    return (b["qg"], b["k"], b["v"], b["qn"], b["kn"], b["pos"], cache or cache_of(),
            batch or batch_of(), heads, n_dims, *sections, theta, 1e-6, b["qo"], b["go"])


def attend(cache=None, batch=None, heads=8, f16=False, tokens=7, d=256, **over):
    size = 2 if f16 else 4
    b = dict(q=fake(size * tokens * heads * d), g=fake(4 * tokens * heads * d),
             o=fake(size * tokens * heads * d))
    b.update(over)
    gate = [] if f16 else [b["g"]]
    return (b["q"], *gate, cache or cache_of(), batch or batch_of(), heads, b["o"])


CACHE_ERRORS = [
    (dict(pages=0), "dimensions must be positive"),
    (dict(pt=48), "pages of 16/32/64/128 tokens"),
    (dict(pt=8), "pages of 16/32/64/128 tokens"),
    (dict(d=192), "supports head_dim 64/128/256"),
    (dict(kp=fake(5 * 64 * 2 * 256 - 1)), "key pages buffer is too small"),
    (dict(vp=kh.KrakenBuffer(None, 1 << 30)), "value pages buffer is not initialized"),
    (dict(ks=fake(39)), "key scales buffer is too small"),
    (dict(vs=fake(0)), "value scales buffer is too small"),
    (dict(kp=fake(1 << 30, 0x1008)), "pages must be 16-byte aligned"),
    (dict(pages=1 << 61), "page count exceeds int32 range"),
]
BATCH_ERRORS = [
    (dict(sequences=0), "batch dimensions must be positive"),
    (dict(max_query=0), "batch dimensions must be positive"),
    (dict(tokens=0), "batch dimensions must be positive"),
    (dict(max_keys=1 << 31), "batch exceeds int32 range"),
    (dict(sequences=(1 << 19) + 1), "takes up to 1048576 pairs"),
    (dict(width=1 << 62), "overflow"),
    (dict(table=fake(23)), "page table buffer is too small"),
    (dict(starts=fake(12)), "query starts buffer is too small"),
    (dict(lengths=kh.KrakenBuffer(None, 64)), "lengths buffer is not initialized"),
]


@pytest.mark.parametrize("kw,fragment", CACHE_ERRORS)
def test_cache_refusals(vctx, kw, fragment):
    for name, args in (("qwen35_attention_prologue_paged_q8_kv", prologue(cache=cache_of(**kw))),
                       ("attention_f32_paged_q8_kv", attend(cache=cache_of(**kw))),
                       ("attention_f16q_paged_q8_kv", attend(cache=cache_of(**kw), f16=True)),
                       ("dequantize_kv_pages_q8_f16",
                        (cache_of(**kw), fake(4), 1, fake(1 << 20), fake(1 << 20)))):
        assert vctx.status(name, *args) == kh.INVALID_ARGUMENT
        assert fragment in kh.last_error(), (name, kh.last_error())


@pytest.mark.parametrize("kw,fragment", BATCH_ERRORS)
def test_batch_refusals(vctx, kw, fragment):
    for name, args in (("qwen35_attention_prologue_paged_q8_kv", prologue(batch=batch_of(**kw))),
                       ("attention_f32_paged_q8_kv", attend(batch=batch_of(**kw))),
                       ("attention_f16q_paged_q8_kv", attend(batch=batch_of(**kw), f16=True))):
        assert vctx.status(name, *args) == kh.INVALID_ARGUMENT
        assert fragment in kh.last_error(), (name, kh.last_error())


@pytest.mark.parametrize("kw,fragment", [
    (dict(heads=0), "dimensions must be positive"),
    (dict(heads=3), "divisible by kv_heads"),
    (dict(n_dims=63), "MRoPE dimensions are invalid"),
    (dict(n_dims=258), "MRoPE dimensions are invalid"),
    (dict(sections=(0, 0, 0, 0)), "sections must not all be zero"),
    (dict(theta=0.0), "theta must be positive"),
    (dict(theta=math.inf), "theta must be positive"),
    (dict(qg=fake(8 * 7 * 8 * 256 - 4)), "q_gate buffer is too small"),
    (dict(v=fake(16)), "value buffer is too small"),
    (dict(kn=kh.KrakenBuffer(None, 4096)), "k_norm buffer is not initialized"),
    (dict(pos=fake(111)), "positions buffer is too small"),
    (dict(go=fake(4)), "gate output buffer is too small"),
])
def test_prologue_refusals(vctx, kw, fragment):
    assert vctx.status("qwen35_attention_prologue_paged_q8_kv",
                       *prologue(**kw)) == kh.INVALID_ARGUMENT
    assert fragment in kh.last_error()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("kw,fragment", [
    (dict(heads=0), "dimensions must be positive"),
    (dict(heads=5), "divisible by kv_heads"),
    (dict(q=fake(64)), "query buffer is too small"),
    (dict(o=kh.KrakenBuffer(None, 1 << 20)), "output buffer is not initialized"),
    (dict(q=fake(1 << 20, 0x1004)), "buffers must be 16-byte aligned"),
    (dict(batch=batch_of(tokens=(1 << 31) - 1), o=fake(1 << 62), q=fake(1 << 62)),
     "takes up to 67108864 query rows"),
])
def test_attention_refusals(vctx, kw, fragment, f16):
    name = "attention_f16q_paged_q8_kv" if f16 else "attention_f32_paged_q8_kv"
    assert vctx.status(name, *attend(f16=f16, **kw)) == kh.INVALID_ARGUMENT
    assert fragment in kh.last_error()


def test_gate_refusal_and_null_structs(vctx):
    assert vctx.status("attention_f32_paged_q8_kv", *attend(g=fake(8))) == kh.INVALID_ARGUMENT
    assert "gate buffer is too small" in kh.last_error()
    q, g, _, batch, heads, o = attend()
    assert vctx.status("attention_f32_paged_q8_kv", q, g, None, batch, heads,
                       o) == kh.INVALID_ARGUMENT
    assert "cache must not be null" in kh.last_error()
    assert vctx.status("attention_f32_paged_q8_kv", q, g, cache_of(), None, heads,
                       o) == kh.INVALID_ARGUMENT
    assert "batch must not be null" in kh.last_error()


def test_accepted(vctx):
    no = kh.KrakenBuffer(None, 0)
    for name, args in (
            ("qwen35_attention_prologue_paged_q8_kv", prologue()),
            ("qwen35_attention_prologue_paged_q8_kv", prologue(pos=no)),
            ("attention_f32_paged_q8_kv", attend()), ("attention_f32_paged_q8_kv", attend(g=no)),
            ("attention_f16q_paged_q8_kv", attend(f16=True)),
            ("dequantize_kv_pages_q8_f16",
             (cache_of(), fake(8), 2, fake(4 * 64 * 512), fake(4 * 64 * 512))),
            ("sample_f32_i32", (fake(4 * 25), 3, 5, 10, no, no, no, no, fake(12), fake(12), no))):
        assert vctx.status(name, *args) == kh.UNAVAILABLE, (name, kh.last_error())
        assert kh.last_error() == ACCEPTED


def test_dequantize_refusals(vctx):
    rows = fake(4 * 64 * 512)
    for args, fragment in (((cache_of(), fake(8), 0, rows, rows), "dimensions must be positive"),
                           ((cache_of(), fake(7), 2, rows, rows), "page ids buffer is too small"),
                           ((cache_of(), fake(8), 2, fake(64), rows), "key rows buffer is too small"),
                           ((cache_of(), fake(1 << 40), 1 << 30, fake(1 << 60), fake(1 << 60)),
                            "too many pages at once"),
                           ((cache_of(), fake(8), 2, rows, fake(4 * 64 * 512, 0x1002)),
                            "rows must be 16-byte aligned")):
        assert vctx.status("dequantize_kv_pages_q8_f16", *args) == kh.INVALID_ARGUMENT
        assert fragment in kh.last_error()


def test_sample_refusals(vctx):
    no = kh.KrakenBuffer(None, 0)
    base = [fake(4 * 25), 3, 5, 10, no, no, no, no, fake(12), fake(12), fake(12)]
    for at, value, fragment in ((1, 0, "dimensions must be positive"),
                                (2, 0, "dimensions must be positive"),
                                (3, 4, "row stride must be at least the row size"),
                                (0, fake(4 * 25 - 4), "logits buffer is too small"),
                                (3, 1 << 62, "overflow"),
                                (4, fake(8), "temperature buffer is too small"),
                                (5, fake(8), "top_k buffer is too small"),
                                (6, fake(8), "top_p buffer is too small"),
                                (7, fake(8), "min_p buffer is too small"),
                                (8, no, "uniforms buffer is not initialized"),
                                (9, fake(8), "token output buffer is too small"),
                                (10, fake(8), "probability output buffer is too small")):
        args = list(base)
        args[at] = value
        assert vctx.status("sample_f32_i32", *args) == kh.INVALID_ARGUMENT
        assert fragment in kh.last_error(), kh.last_error()
    for rows, size in ((1, (1 << 22) + 1), (65536, 5)):
        args = list(base)
        args[0], args[1], args[2], args[3] = fake(1 << 40), rows, size, size
        assert vctx.status("sample_f32_i32", *args) == kh.INVALID_ARGUMENT
        assert "rows of up to 4194304 logits" in kh.last_error()


# ------------------------------------------------------- the plain forms ----


def test_plain_append_growth_stays_within_one_step():
    """Rows that grow 2.3 times each: the first row ends within a step of itself."""
    rng = np.random.default_rng(3)
    cache = po.Pages(rng, 1, 16, 1, 64)
    rows = rng.standard_normal((16, 1, 64)) * (2.3 ** np.arange(16))[:, None, None]
    table = np.zeros((1, 1), np.int32)
    for i in range(16):
        po.append(cache, "key", rows[i:i + 1], (table, [0, 1], [i + 1], 1, 1, 16))
    got, step = cache.values_of("key", 0)[:, 0], float(cache.scales["key"][0, 0])
    assert np.abs(got - rows[:, 0]).max() <= step
    assert np.abs(rows).max() <= 127.0 * step <= 2.0 * np.abs(rows).max()


def test_plain_append_fresh_page_is_half_a_step_off():
    rng = np.random.default_rng(4)
    cache = po.Pages(rng, 2, 16, 2, 64)
    rows = rng.standard_normal((20, 2, 64))
    po.append(cache, "value", rows, (np.array([[1, 0]], np.int32), [0, 20], [20], 20, 20, 32))
    got = np.concatenate([cache.values_of("value", 1), cache.values_of("value", 0)[:4]])
    for page, span in ((1, slice(0, 16)), (0, slice(16, 20))):
        steps = cache.scales["value"][page].astype(np.float64)
        assert (np.abs(got[span] - rows[span]) <= (0.5 + 1e-5) * steps[None, :, None]).all()


def test_plain_rotation_is_a_complex_rotation():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 2, 64))
    pos = np.array([[5, 0, 100003]] * 4)
    y = po.norm_rope(x, np.ones(64), pos, 64, (11, 11, 10, 0), 1e4, 0.0)
    unit = x / np.sqrt((x * x).mean(-1, keepdims=True))
    z = (unit[..., :32] + 1j * unit[..., 32:])
    z = z * np.exp(1j * pos[0][:, None, None] * 1e4 ** (-np.arange(32) / 32))
    np.testing.assert_allclose(y, np.concatenate([z.real, z.imag], -1), rtol=0, atol=1e-9)


def test_plain_attention_closed_forms():
    """A zero query takes the mean of its keys' values; the first position its own."""
    rng = np.random.default_rng(6)
    cache = po.Pages(rng, 3, 16, 1, 64)
    batch = (np.array([[2, 0]], np.int32), [0, 3], [19], 3, 3, 32)
    out, _, _ = po.attention(cache, np.zeros((3, 2, 64)), batch, 2)
    v = np.concatenate([cache.values_of("value", 2), cache.values_of("value", 0)])[:, 0]
    for i in range(3):
        np.testing.assert_allclose(out[i], np.broadcast_to(v[:17 + i].mean(0), (2, 64)), rtol=1e-12)
    out, _, _ = po.attention(cache, rng.standard_normal((1, 2, 64)),
                             (np.array([[2, 0]], np.int32), [0, 1], [1], 1, 1, 32), 2)
    np.testing.assert_allclose(out[0], np.broadcast_to(v[0], (2, 64)), rtol=1e-12)


def test_plain_sample_known_answers():
    x = np.log([0.1, 0.4, 0.2, 0.3])
    # Index order: 0.1, 0.5, 0.7, 1.0.
    assert [po.sample(x, uniform=u)[0] for u in (0.05, 0.3, 0.6, 0.9)] == [0, 1, 2, 3]
    assert po.sample(x, top_k=2, uniform=0.5)[0] == 1  # 0.4 / 0.7 above a half
    assert po.sample(x, top_k=2, uniform=0.6)[0] == 3
    assert po.sample(x, top_p=0.65, uniform=0.999)[0] == 3
    np.testing.assert_allclose(po.sample(x, top_p=0.65, uniform=0.999)[1], 3 / 7)
    assert po.sample(x, min_p=0.6, uniform=0.1)[0] == 1
    assert po.sample(x, temperature=0.0, uniform=0.99) == (1, 1.0)
    assert po.sample([1.0, 1.0, 1.0, 1.0], top_k=2, uniform=0.9)[0] == 1
    assert po.sample([math.nan, -math.inf], uniform=0.5) == (1, 0.0)
    assert po.sample([math.nan] * 3, uniform=0.5) == (3, 0.0)
    assert po.sample([0.0, math.inf, 1.0, math.inf], uniform=0.6) == (3, 0.5)
