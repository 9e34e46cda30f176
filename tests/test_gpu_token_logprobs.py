"""token_logprobs_f32 on the GPU against the plain 64-bit form (tests/serving_oracle.py,
which derives the tolerances).  Tokens and ranks are equal."""
import math

import numpy as np
import pytest

import kraken_hip as kh
import serving_oracle as so

pytestmark = pytest.mark.gpu


def run(ctx, logits, tokens, top, temperature=None, stride=None, entropy=True):
    rows, size = logits.shape
    stride = stride or size
    padded = np.full((rows, stride), 90.0, np.float32)
    padded[:, :size] = logits
    outs = {"logprob": np.full(rows, 7, np.float32), "rank": np.full(rows, -7, np.int32),
            "entropy": np.full(rows, 7, np.float32),
            "top_tokens": np.full((rows, top), -7, np.int32),
            "top_logprobs": np.full((rows, top), 7, np.float32)}
    bufs = {n: ctx.buffer(x) for n, x in outs.items()}
    given = None if tokens is None else ctx.buffer(np.asarray(tokens, np.int32))
    t = None if temperature is None else ctx.buffer(np.asarray(temperature, np.float32))
    ctx.token_logprobs_f32(ctx.buffer(padded), rows, size, stride, t, given, top,
                           bufs["logprob"] if given else None, bufs["rank"] if given else None,
                           bufs["entropy"] if entropy else None,
                           bufs["top_tokens"] if top else None,
                           bufs["top_logprobs"] if top else None)
    return {n: b.download(outs[n].size).reshape(outs[n].shape) for n, b in bufs.items()}


def close(got, want, off):
    # Past f32's largest (3.4028236e38 with half a step) a value rounds to infinity.
    if not math.isfinite(want) or abs(want) > 3.4028236e38:
        return got == math.copysign(math.inf, want)
    return abs(float(got) - want) <= off


def check(ctx, logits, tokens, top, temperature=None, stride=None):
    logits = np.asarray(logits, np.float32)
    got = run(ctx, logits, tokens, top, temperature, stride)
    for r, row in enumerate(logits):
        t = 1.0 if temperature is None else float(np.float32(temperature[r]))
        want = so.logprobs(row, t, int(tokens[r]), top)
        assert got["rank"][r] == want["rank"], (r, got["rank"][r], want["rank"])
        assert got["top_tokens"][r].tolist() == want["top_tokens"], r
        for n, off in (("logprob", "logprob_off"), ("entropy", "entropy_off")):
            assert close(got[n][r], want[n], want[off]), (r, n, got[n][r], want[n], want[off])
        for i in range(top):
            assert close(got["top_logprobs"][r, i], want["top_logprobs"][i], want["top_off"][i]), (
                r, i, got["top_logprobs"][r, i], want["top_logprobs"][i])
    return got


@pytest.mark.parametrize("size", [1, 2, 3, 5, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 8191,
                                  8193, 32003, 151936, 248320])
@pytest.mark.parametrize("spread", [0.3, 3.0, 30.0])
def test_matches_plain(hip_ctx, size, spread):
    rng = np.random.default_rng(size)
    rows = 7 if size < 40000 else 3
    logits = (spread * rng.standard_normal((rows, size))).astype(np.float32)
    for top in (1, 5, 32):
        temperature = rng.choice([0.3, 0.7, 1.0, 2.5, 0.0, -1.0, math.nan], rows)
        check(hip_ctx, logits, rng.integers(0, size, rows), top, temperature, size + top % 3)


def test_likeliest_token_takes_nearly_everything(hip_ctx):
    """Log probabilities and entropies near zero keep their relative accuracy."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((6, 50000)).astype(np.float32)
    at = rng.integers(0, 50000, 6)
    for r, lead in enumerate((12.0, 20.0, 30.0, 45.0, 70.0, 100.0)):
        logits[r, at[r]] = lead
    got = check(hip_ctx, logits, at, 4)
    assert (got["logprob"][:5] < 0).all() and (got["rank"] == 0).all()


@pytest.mark.parametrize("size", [7, 300, 5000, 70000])
def test_ties_and_values_out_of_the_ordinary(hip_ctx, size):
    """Equal logits, masked vocabularies, NaN and infinities, few or none left."""
    rng = np.random.default_rng(size)
    rows = []
    rows.append(np.zeros(size))
    rows.append(rng.integers(0, 3, size).astype(float))
    masked = np.full(size, -math.inf)
    masked[[size // 2, size - 1]] = (1.0, 2.0)
    rows += [masked, np.full(size, -math.inf), np.full(size, math.nan)]
    some = rng.standard_normal(size)
    some[::2] = math.nan
    some[1] = -math.inf
    rows.append(some)
    two = rng.standard_normal(size)
    two[[2, size - 2]] = math.inf
    rows.append(two)
    rows.append(np.where(rng.random(size) < 0.5, -3.4e38, 3.4e38))
    rows.append(np.full(size, np.finfo(np.float32).min))
    rows.append(rng.choice([-0.0, 0.0, 1e-40, -1e-40], size))
    lowest = rng.standard_normal(size)
    lowest[: size // 2] = np.finfo(np.float32).min  # a mask of the type's lowest value
    rows.append(lowest)
    mixed = np.where(rng.random(size) < 0.5, math.nan, -math.inf)
    rows.append(mixed)
    logits = np.array(rows, np.float32)
    n = len(rows)
    for tokens in (rng.integers(0, size, n), np.zeros(n, int), np.full(n, size - 1),
                   rng.choice([-1, size, 2 ** 31 - 1, -2 ** 31, 1], n)):
        for temperature in (None, np.full(n, 0.7), np.full(n, 1e-30), np.full(n, 1e30)):
            check(hip_ctx, logits, tokens, 9, temperature)


def test_infinite_and_least_temperatures(hip_ctx):
    """Beyond f32's quotients: all real logits alike, and the largest alone."""
    logits = np.array([[1.0, 3.0, -math.inf, 2.0, 3.0], [0.0, -1.0, math.nan, 5.0, 4.0]], np.float32)
    got = check(hip_ctx, logits, [0, 1], 5, [math.inf, math.inf])
    np.testing.assert_allclose(got["logprob"], -math.log(4), rtol=1e-6)
    got = check(hip_ctx, logits, [1, 3], 5, [1e-45, 1e-45])
    np.testing.assert_allclose(got["logprob"], [-math.log(2), 0.0], rtol=1e-6)


def test_sorted_rows_and_one_thread_s_share(hip_ctx):
    """The largest side by side, or so far apart that one thread holds them all."""
    size = 40000
    rows = [np.arange(size), -np.arange(size)]
    for step in (16, 64, 256, 1024):
        x = np.random.default_rng(step).standard_normal(size)
        x[:step * 32:step] += 100.0
        rows.append(x)
    check(hip_ctx, np.array(rows, np.float32) / 50.0, np.arange(len(rows)), 32)


def test_each_output_alone(hip_ctx):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((3, 3001)).astype(np.float32)
    whole = run(hip_ctx, logits, [5, 6, 7], 3)
    only = run(hip_ctx, logits, None, 3, entropy=False)
    assert (only["logprob"] == 7).all() and (only["rank"] == -7).all()
    assert (only["entropy"] == 7).all()
    for n in ("top_tokens", "top_logprobs"):
        np.testing.assert_array_equal(only[n], whole[n])
    for n in ("logprob", "rank", "entropy"):
        rest = run(hip_ctx, logits, [5, 6, 7], 0)
        np.testing.assert_array_equal(rest[n], whole[n])


def test_many_rows_and_their_alignment(hip_ctx):
    """More rows than run at once; a row stride that leaves rows misaligned."""
    rng = np.random.default_rng(6)
    logits = (2 * rng.standard_normal((700, 900))).astype(np.float32)
    check(hip_ctx, logits, rng.integers(0, 900, 700), 2, stride=901)
    torch = pytest.importorskip("torch")
    x = torch.zeros(65535, 3, device="cuda")
    x[:, 1] = 1.0
    out = torch.zeros(65535, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    hip_ctx.token_logprobs_f32(x, 65535, 3, 3, None, None, 1, None, None, None, out, None)
    assert bool((out == 1).all())


def test_the_same_bits_in_any_batch_and_replay(hip_ctx):
    """A row's outputs do not depend on its neighbours, and a captured call replays."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(7)
    logits = (3 * rng.standard_normal((40, 20000))).astype(np.float32)
    tokens = rng.integers(0, 20000, 40)
    whole = run(hip_ctx, logits, tokens, 20)
    for r in (0, 17, 39):
        one = run(hip_ctx, logits[r:r + 1], tokens[r:r + 1], 20)
        for n, x in one.items():
            np.testing.assert_allclose(x[0], whole[n][r], rtol=0 if x.dtype.kind == "i" else 1e-6)
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    sets = [torch.from_numpy((2 * rng.standard_normal((5, 9000))).astype(np.float32)).cuda()
            for _ in range(3)]
    t = torch.tensor([1, 2, 3, 4, 5], dtype=torch.int32, device="cuda")

    def outputs():
        return [torch.zeros(5, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"),
                torch.zeros(5, device="cuda"),
                torch.zeros(5, 7, dtype=torch.int32, device="cuda"),
                torch.zeros(5, 7, device="cuda")]

    x, got, want = sets[0].clone(), outputs(), outputs()
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ctx.token_logprobs_f32(x, 5, 9000, 9000, None, t, 7, *got)
        for s in sets:
            x.copy_(s)
            graph.replay()
            ctx.token_logprobs_f32(s, 5, 9000, 9000, None, t, 7, *want)
            stream.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    ctx.commit_graph()
    ctx.close()


@pytest.mark.parametrize("size,places,chunks", [
    (4096, 124, 1), (4096, 128, 1), (9000, 124, 2), (40000, 128, 9), (200000, 128, 45),
    (700000, 128, 170)])
def test_top_places_that_crowd(hip_ctx, size, places, chunks):
    """The largest logits in the same places of every 256 of a chunk of 4096: more candidates
    than threads, in a chunk and over all chunks, and a list that rises from chunk to chunk."""
    rng = np.random.default_rng(size + places)
    rows = rng.standard_normal((3, size))
    at = np.arange(size)
    crowd = at % 256 < places
    rows[0, crowd] += 100.0
    # 28 in half of the chunks, by eights.
    rows[1, (at // 4096 % 8 < 4) & (at % 4096 < 28)] += 100.0
    rows[2] = at * 1e-4
    assert -(-size // 4096) >= chunks
    for top in (32, 20, 1):
        check(hip_ctx, rows, rng.integers(0, size, 3), top)


def test_single_outputs(hip_ctx):
    """Each output alone is what it is among all."""
    rng = np.random.default_rng(9)
    rows, size, top = 5, 9001, 7
    logits = hip_ctx.buffer((3 * rng.standard_normal((rows, size))).astype(np.float32))
    tokens = hip_ctx.buffer(rng.integers(0, size, rows).astype(np.int32))

    def outs():
        return [hip_ctx.buffer(np.full(rows * n, -7, k)) for n, k in
                ((1, np.float32), (1, np.int32), (1, np.float32), (top, np.int32), (top, np.float32))]

    def call(bufs):
        hip_ctx.token_logprobs_f32(logits, rows, size, size, None,
                                   tokens if bufs[0] or bufs[1] else None,
                                   top if bufs[3] or bufs[4] else 0, *bufs)

    everything = outs()
    call(everything)
    for i in range(5):
        one = [b if j == i else None for j, b in enumerate(outs())]
        call(one)
        np.testing.assert_array_equal(one[i].download(dtype=np.int32),
                                      everything[i].download(dtype=np.int32))
