"""A captured batched step whose replays bring other batches: sequences that move between
single tokens and chunks, so that their rows move between the kernels of few and of many
rows, and lengths that make the tiled kernel choose other parts.  Each replay equals the
eager calls bit by bit and the plain form to the tolerance of tests/test_gpu_paged_q8.py.
"""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po

pytestmark = pytest.mark.gpu

# (new tokens, tokens before) of each sequence, replay by replay.
SEVERAL = [([160, 1, 4, 5], [0, 900, 33, 70]), ([1, 150, 17, 0], [40, 2900, 0, 5]),
           ([4, 4, 4, 4], [3000, 10, 500, 64]), ([5, 3, 1, 150], [2900, 1, 700, 1500]),
           ([1, 1, 1, 1], [0, 15, 16, 3000]), ([60, 60, 60, 1], [2000, 0, 1000, 31])]
# Of 1360 tiles' parts of 128 keys each, more than run at once, and of fewer.
LONG = [([160, 100, 1], [6000, 3000, 10]), ([5, 1, 1], [6000, 0, 100]),
        ([8, 160, 90], [0, 1000, 60]), ([160, 160, 2], [300, 5900, 6000])]
ONE = [([150], [1000]), ([1], [3000]), ([8], [0]), ([9], [77]), ([160], [2900]), ([0], [50])]


class Step:
    """The device arrays of a step and its calls."""

    def __init__(self, torch, cache, sequences, width, tokens, max_query, max_keys, heads, f16):
        self.torch, self.cache, self.heads, self.f16 = torch, cache, heads, f16
        d, kv = cache.head_dim, cache.kv_heads
        self.shape = (tokens, heads, d)
        kind = torch.float16 if f16 else torch.float32
        self.t = {"keys": torch.from_numpy(cache.codes["key"]).cuda(),
                  "values": torch.from_numpy(cache.device_values()).cuda(),
                  "ks": torch.from_numpy(cache.scales["key"]).cuda(),
                  "vs": torch.from_numpy(cache.scales["value"]).cuda(),
                  "table": torch.zeros(sequences, width, dtype=torch.int32, device="cuda"),
                  "starts": torch.zeros(sequences + 1, dtype=torch.int32, device="cuda"),
                  "lengths": torch.zeros(sequences, dtype=torch.int32, device="cuda"),
                  "qg": torch.zeros(tokens, heads, 2 * d, device="cuda"),
                  "k": torch.zeros(tokens, kv, d, device="cuda"),
                  "v": torch.zeros(tokens, kv, d, device="cuda"),
                  "w": torch.ones(d, device="cuda"),
                  "q": torch.zeros(self.shape, device="cuda"),
                  "g": torch.zeros(self.shape, device="cuda"),
                  "half": torch.zeros(self.shape, device="cuda", dtype=torch.float16),
                  "out": torch.zeros(self.shape, device="cuda", dtype=kind)}
        b = {n: kh.as_buffer(x) for n, x in self.t.items()}
        self.pages = kh.PagedQ8Cache(b["keys"], b["values"], b["ks"], b["vs"], cache.pages,
                                     cache.page_tokens, kv, d)
        self.batch = kh.PagedBatch(b["table"], b["starts"], b["lengths"], sequences, width, tokens,
                                   max_query, max_keys)

    def set(self, arrays):
        for n, x in arrays.items():
            self.t[n].copy_(self.torch.from_numpy(x))
        self.t["out"].fill_(-77)
        self.t["q"].fill_(-77)

    def run(self, ctx):
        t = self.t
        ctx.qwen35_attention_prologue_paged_q8_kv(
            t["qg"], t["k"], t["v"], t["w"], t["w"], None, self.pages, self.batch, self.heads, 64,
            11, 11, 10, 0, 1e7, 1e-6, t["q"], t["g"])
        if self.f16:
            t["half"].copy_(t["q"])
            ctx.attention_f16q_paged_q8_kv(t["half"], self.pages, self.batch, self.heads, t["out"])
        else:
            ctx.attention_f32_paged_q8_kv(t["q"], t["g"], self.pages, self.batch, self.heads,
                                          t["out"])


def arrays_of(rng, cache, new, before, width, tokens, heads):
    lengths = [a + b for a, b in zip(new, before)]
    table = np.full((len(new), width), -1, np.int32)
    order, at = rng.permutation(cache.pages), 0
    for b, length in enumerate(lengths):
        n = -(-length // cache.page_tokens)
        table[b, :n] = order[at:at + n]
        at += n
    d, kv = cache.head_dim, cache.kv_heads
    return {"table": table, "starts": np.concatenate([[0], np.cumsum(new)]).astype(np.int32),
            "lengths": np.array(lengths, np.int32),
            "qg": (2 * rng.standard_normal((tokens, heads, 2 * d))).astype(np.float32),
            "k": rng.standard_normal((tokens, kv, d)).astype(np.float32),
            "v": rng.standard_normal((tokens, kv, d)).astype(np.float32)}


def plain_rows(held, query, gate, arrays, heads, rows):
    """(output, magnitude, score) of single rows of the batch."""
    starts, lengths = arrays["starts"].astype(np.int64), arrays["lengths"].astype(np.int64)
    found = []
    for r in rows:
        b = int(np.searchsorted(starts[1:], r, side="right"))
        length = int(lengths[b] - (starts[b + 1] - 1 - r))
        one = (arrays["table"][b:b + 1], np.array([0, 1]), np.array([length]), 1, 1, length)
        found.append(po.attention(held, query[r:r + 1], one, heads,
                                  None if gate is None else gate[r:r + 1]))
    return [np.concatenate(x) for x in zip(*found)]


@pytest.mark.parametrize("batches,f16,d,heads,kv,pt", [
    *[(b, *kind) for b in (SEVERAL, ONE) for kind in ((False, 128, 8, 2, 16), (True, 64, 6, 1, 64),
                                                      (False, 256, 4, 1, 32))],
    (LONG, False, 64, 16, 4, 128), (LONG, True, 128, 16, 4, 64)])
def test_replays_of_other_batches(hip_ctx, batches, f16, d, heads, kv, pt):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(d + len(batches[0][0]))
    tokens = max(sum(new) for new, _ in batches) + 1
    max_query = max(max(new) for new, _ in batches)
    longest = max(a + b for new, before in batches for a, b in zip(new, before))
    width = -(-longest // pt)
    most = max(sum(-(-(a + b) // pt) for a, b in zip(new, before)) for new, before in batches)
    cache = po.Pages(rng, most + 2, pt, kv, d)
    steps = [Step(torch, cache, len(batches[0][0]), width, tokens, max_query, longest, heads, f16)
             for _ in range(2)]
    eager, captured = steps
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured.run(ctx)
        for i, (new, before) in enumerate(batches + batches[:2]):
            arrays = arrays_of(rng, cache, new, before, width, tokens, heads)
            for s in steps:
                s.set(arrays)
            graph.replay()
            eager.run(ctx)
            stream.synchronize()
            for n in ("keys", "values", "ks", "vs", "q", "out"):
                assert torch.equal(eager.t[n], captured.t[n]), (i, n)
            held = po.Pages.__new__(po.Pages)
            held.__dict__.update(cache.__dict__)
            shape = cache.codes["key"].shape
            held.codes = {"key": captured.t["keys"].cpu().numpy(),
                          "value": np.empty(shape, np.int8)}
            held.set_device_values(captured.t["values"].cpu().numpy())
            held.scales = {"key": captured.t["ks"].cpu().numpy(),
                           "value": captured.t["vs"].cpu().numpy()}
            query = captured.t["half" if f16 else "q"].cpu().numpy()
            gate = None if f16 else captured.t["g"].cpu().numpy()
            used = sum(new)
            rows = np.arange(used)
            if batches is LONG:
                rows = np.unique(np.concatenate([rng.integers(0, used, 20), arrays["starts"][:-1],
                                                 arrays["starts"][1:] - 1]))
            got = captured.t["out"].cpu().numpy().astype(np.float64)
            assert (got[used:] == -77).all(), i
            if used == 0:
                continue
            want, size, score = plain_rows(held, query, gate, arrays, heads, rows)
            tol = po.attention_tolerance(size, want, score, d, f16)
            off = np.abs(got[rows] - want) / tol
            assert (off <= 1).all(), (i, float(off.max()))
    ctx.commit_graph()
    ctx.close()
