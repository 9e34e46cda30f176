"""sample_f32_i32 on the GPU against the plain 64-bit form (tests/paged_oracle.py).

Tokens are equal.  The kernel's weights are integers of 2^-44 of the largest or finer,
so a draw could differ only where the uniform falls within about 1e-10 of a border; the
uniforms are drawn, or placed well inside a token's share.  A probability is the
quotient of two sums rounded once to f32 (half a step, 2^-24), and the sums' own
rounding is below another: 2^-23 relative.
"""
import math

import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po

pytestmark = pytest.mark.gpu


def run(ctx, logits, uniforms, stride=None, **rules):
    rows, size = logits.shape
    stride = stride or size
    padded = np.full((rows, stride), 50.0, np.float32)
    padded[:, :size] = logits
    tokens = ctx.buffer(np.full(rows, -7, np.int32))
    share = ctx.buffer(np.full(rows, -7, np.float32))
    kinds = {"temperature": np.float32, "top_k": np.int32, "top_p": np.float32,
             "min_p": np.float32}
    bufs = [ctx.buffer(np.asarray(rules[n], k)) if n in rules else None for n, k in kinds.items()]
    ctx.sample_f32_i32(ctx.buffer(padded), rows, size, stride, *bufs,
                       ctx.buffer(np.asarray(uniforms, np.float32)), tokens, share)
    return tokens.download(dtype=np.int32), share.download()


def check(ctx, logits, uniforms, stride=None, **rules):
    logits = np.asarray(logits, np.float32)
    got, share = run(ctx, logits, uniforms, stride, **rules)
    for r in range(len(logits)):
        rule = {n: v[r] for n, v in rules.items()}
        token, p = po.sample(logits[r], uniform=uniforms[r], **rule)
        assert got[r] == token, (r, rule, uniforms[r], got[r], token)
        assert abs(share[r] - p) <= 2.0 ** -23 * p + 2.0 ** -140, (r, rule, share[r], p)
    return got


def rules_of(rng, rows):
    return {"temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.6], rows).astype(np.float32),
            "top_k": rng.choice([0, 1, 2, 7, 50, 1000, 1 << 30, -3], rows).astype(np.int32),
            "top_p": rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 2.0], rows).astype(np.float32),
            "min_p": rng.choice([0.0, 0.0, 0.01, 0.3, 1.0], rows).astype(np.float32)}


@pytest.mark.parametrize("size", [1, 2, 3, 63, 64, 65, 1000, 1024, 1025, 4096, 4097, 32003, 151936])
@pytest.mark.parametrize("spread", [0.2, 3.0])
def test_sample_matches_plain(hip_ctx, size, spread):
    rng = np.random.default_rng(size)
    rows = 13 if size < 40000 else 5
    logits = (spread * rng.standard_normal((rows, size))).astype(np.float32)
    check(hip_ctx, logits, rng.random(rows).astype(np.float32), **rules_of(rng, rows))


@pytest.mark.parametrize("name,values", [
    ("temperature", [0.5, 1e-4, 3.0, math.inf]), ("top_k", [1, 5, 300, 4999]),
    ("top_p", [0.0, 0.3, 0.8, 0.9999]), ("min_p", [0.001, 0.1, 0.9, 1.5])])
def test_each_rule_alone(hip_ctx, name, values):
    rng = np.random.default_rng(len(name))
    logits = (2 * rng.standard_normal((len(values), 5000))).astype(np.float32)
    check(hip_ctx, logits, rng.random(len(values)).astype(np.float32), **{name: values})


def test_no_rules_and_a_row_stride(hip_ctx):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((3, 777)).astype(np.float32)
    check(hip_ctx, logits, rng.random(3).astype(np.float32))
    check(hip_ctx, logits, rng.random(3).astype(np.float32), stride=1001)


def test_the_full_vocabulary(hip_ctx):
    rng = np.random.default_rng(6)
    logits = (2.5 * rng.standard_normal((6, 248320))).astype(np.float32)
    logits[np.arange(6), rng.integers(0, 248320, 6)] += 9.0
    check(hip_ctx, logits, rng.random(6).astype(np.float32),
          temperature=[1.0, 0.7, 1.0, 0.9, 1.0, 2.0], top_k=[0, 40, 0, 100000, 0, 0],
          top_p=[1.0, 0.95, 0.9, 0.8, 0.9999, 0.5], min_p=[0.0, 0.0, 0.02, 0.0, 0.0, 0.0])


def test_ties(hip_ctx):
    """Equal logits: a cut inside them keeps the lower indices."""
    rng = np.random.default_rng(7)
    flat = np.zeros((5, 3000), np.float32)
    u = np.array([0.0, 0.2, 0.5004, 0.77, 0.9999], np.float32)
    check(hip_ctx, flat, u)
    check(hip_ctx, flat, u, top_k=[1, 10, 1500, 2999, 3000])
    check(hip_ctx, flat, u, top_p=[0.1004, 0.25004, 0.5004, 0.9004, 0.33304])
    few = rng.integers(0, 4, (5, 3000)).astype(np.float32)
    few[:, ::7] = -0.0
    few[:, 3::7] = 0.0
    check(hip_ctx, few, u, top_k=[5, 700, 800, 1700, 2500], top_p=[0.5, 0.9, 0.7, 0.99, 0.3])


def test_flat_rows_of_the_full_vocabulary(hip_ctx):
    """Every logit within a few steps of one value: a cut has all of them to order."""
    rng = np.random.default_rng(8)
    base = np.full((4, 248320), 1.5, np.float32)
    base += rng.integers(0, 40, base.shape).astype(np.float32) * np.float32(2.0 ** -20)
    base[3] = 1.5
    u = rng.random(4).astype(np.float32)
    check(hip_ctx, base, u, top_k=[0, 100000, 70, 1234], top_p=[0.5004, 0.7, 0.9, 0.9])


def test_masked_logits(hip_ctx):
    """-inf, the lowest float, NaN and +inf among the logits, and rows of nothing else."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((9, 2000)).astype(np.float32)
    x[0, :1990] = -np.inf
    x[1, ::2] = np.finfo(np.float32).min
    x[2, ::3] = np.nan
    x[3] = -np.inf
    x[4] = np.nan
    x[5, [7, 99, 1500]] = np.inf
    x[6, 5:] = -np.inf
    x[7, 0] = np.nan
    x[7, 1:] = -np.inf
    x[8] = np.finfo(np.float32).min
    u = rng.random(9).astype(np.float32)
    check(hip_ctx, x, u)
    check(hip_ctx, x, u, temperature=[1e-3] * 9, top_k=[20] * 9, top_p=[0.9] * 9)
    check(hip_ctx, x, u, temperature=[math.inf] * 9, min_p=[0.5] * 9)
    check(hip_ctx, x, u, temperature=[0.0] * 9)


def test_numbers_out_of_range(hip_ctx):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((8, 500)).astype(np.float32)
    u = [0.0, 1.0, 2.0, -1.0, math.nan, 0.5, 0.5, 0.99999994]
    check(hip_ctx, x, u)
    check(hip_ctx, x, u, top_p=[math.nan, 0.5, -1.0, 0.5, 0.5, 0.0, 9.0, 0.7],
          min_p=[math.nan, 0.1, -1.0, 0.1, 0.0, 2.0, 0.0, 0.0],
          temperature=[math.nan, 1.0, 1.0, -2.0, 1.0, 1.0, 1e-45, 1.0])


def test_draws_follow_the_distribution(hip_ctx):
    """A uniform on a fine grid gives each kept token as often as its share says, to
    one draw at each end of it."""
    n = 4096
    x = np.log(np.array([0.1, 0.4, 0.05, 0.3, 0.15], np.float32))
    u = (np.arange(n, dtype=np.float32) + 0.5) / n
    got, share = run(hip_ctx, np.tile(x, (n, 1)), u)
    counts = np.bincount(got, minlength=5)
    assert np.abs(counts - n * np.exp(x)).max() <= 1
    np.testing.assert_allclose(share, np.exp(x)[got], rtol=1e-6)


def test_captured_sampling_replays(hip_ctx):
    """A captured draw replayed with other logits, rules and uniforms equals the eager
    draw each time, with eager calls of another size between."""
    torch = pytest.importorskip("torch")
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    rows, size = 3, 50000
    a = {"x": torch.empty(rows, size, device="cuda"), "u": torch.empty(rows, device="cuda"),
         "p": torch.empty(rows, device="cuda"),
         "k": torch.empty(rows, device="cuda", dtype=torch.int32)}
    out = [torch.empty(rows, device="cuda", dtype=torch.int32) for _ in range(2)]
    share = [torch.empty(rows, device="cuda") for _ in range(2)]
    other = torch.randn(2, 200000, device="cuda")
    other_out = torch.empty(2, device="cuda", dtype=torch.int32)

    def draw(i):
        ctx.sample_f32_i32(a["x"], rows, size, size, None, a["k"], a["p"], None, a["u"], out[i],
                           share[i])

    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            draw(0)
        for seed in range(5):
            torch.manual_seed(seed)
            a["x"].copy_(2 * torch.randn(rows, size))
            a["u"].copy_(torch.rand(rows))
            a["p"].copy_(torch.tensor([0.5, 1.0, 0.99]))
            a["k"].copy_(torch.tensor([0, 1000, 200]))
            graph.replay()
            ctx.sample_f32_i32(other, 2, 200000, 200000, None, None, None, None, a["u"], other_out,
                               None)
            draw(1)
            stream.synchronize()
            assert torch.equal(out[0], out[1]) and torch.equal(share[0], share[1])
    ctx.commit_graph()
    ctx.close()
