"""A server that keeps its sequences within a budget of pages, on the GPU: sequences that
share a prompt's pages append, attend, sum the weight that their keys receive, sample and
score; then each is cut to the keys of most weight, moves into fresh pages and goes on.  Each
step's outputs equal the plain forms (tests/paged_oracle.py, tests/serving_oracle.py) on what
the device held, to their tolerances; eager, and as two captured graphs of one context."""
import numpy as np
import pytest

import kraken_hip as kh
import paged_oracle as po
import serving_oracle as so

pytestmark = pytest.mark.gpu

SIZE, TOP, STRIDE = 1000, 5, 480


class Server:
    def __init__(self, torch, ctx, rng, cache, table, target, lengths, heads):
        self.torch, self.ctx, self.cache, self.heads = torch, ctx, cache, heads
        n, d, kv = len(lengths), cache.head_dim, cache.kv_heads

        def put(x):
            return torch.from_numpy(np.ascontiguousarray(x)).cuda()

        def blank(*shape, kind=torch.float32):
            return torch.zeros(*shape, dtype=kind, device="cuda")

        i32 = torch.int32
        self.t = t = {
            "keys": put(cache.codes["key"]), "values": put(cache.device_values()),
            "ks": put(cache.scales["key"]), "vs": put(cache.scales["value"]),
            "table": put(table), "target": put(target), "lengths": put(lengths),
            "starts": put(np.arange(n + 1, dtype=np.int32)),
            "gs": put(np.array([0, n], np.int32)), "gl": put(np.array([320], np.int32)),
            "positions": blank(4, n, kind=i32), "qg": blank(n, heads, 2 * d),
            "k": blank(n, kv, d), "v": blank(n, kv, d), "norm": torch.ones(d, device="cuda"),
            "q": blank(n, heads, d), "g": blank(n, heads, d), "out": blank(n, heads, d),
            "weights": blank(n, kv, STRIDE), "moved": blank(n, kv, STRIDE),
            "head": put(rng.standard_normal((heads * d, SIZE)).astype(np.float32)),
            "logits": blank(n, SIZE), "uniform": blank(n), "tokens": blank(n, kind=i32),
            "share": blank(n), "logprob": blank(n), "rank": blank(n, kind=i32),
            "entropy": blank(n), "top": blank(n, TOP, kind=i32), "top_logprob": blank(n, TOP),
            "temperature": put(np.array([0.7, 1.0, 1.3, 0.5], np.float32)),
            "keep": blank(n, kind=i32), "counts": blank(n, kind=i32), "kept": blank(n, kv, STRIDE, kind=i32)}
        self.b = {name: kh.as_buffer(x) for name, x in t.items()}
        b, width = self.b, table.shape[1]
        self.pages = kh.PagedQ8Cache(b["keys"], b["values"], b["ks"], b["vs"], cache.pages,
                                     cache.page_tokens, kv, d)
        # (Loose bounds, so that these few keys are shared.)
        self.batch = kh.PagedBatch(b["table"], b["starts"], b["lengths"], n, width, n, 1, 1 << 20)
        self.groups = kh.SharedPrefixes(b["gs"], b["gl"], 1, n, 1 << 20)

    def step(self):
        ctx, t, b, n = self.ctx, self.t, self.b, len(self.t["lengths"])
        t["lengths"].add_(1)
        ctx.qwen35_attention_prologue_paged_q8_kv(
            b["qg"], b["k"], b["v"], b["norm"], b["norm"], b["positions"], self.pages, self.batch,
            self.heads, 64, 11, 11, 10, 0, 1e7, 1e-6, b["q"], b["g"])
        ctx.attention_f32_shared_paged_q8_kv(b["q"], b["g"], self.pages, self.batch, self.groups,
                                             self.heads, b["out"])
        ctx.key_weights_f32_paged_q8_kv(b["q"], self.pages, self.batch, self.heads, 0, 0.9,
                                        b["weights"], STRIDE)
        self.torch.mm(t["out"].view(n, -1), t["head"], out=t["logits"])
        ctx.sample_f32_i32(b["logits"], n, SIZE, SIZE, b["temperature"], None, None, None,
                           b["uniform"], b["tokens"], b["share"])
        ctx.token_logprobs_f32(b["logits"], n, SIZE, SIZE, b["temperature"], b["tokens"], TOP,
                               b["logprob"], b["rank"], b["entropy"], b["top"], b["top_logprob"])

    def evict(self):
        ctx, t, b, n = self.ctx, self.t, self.b, len(self.t["lengths"])
        kv, width = self.cache.kv_heads, t["table"].shape[1]
        ctx.select_keys_f32_i32(b["weights"], STRIDE, b["lengths"], b["keep"], n, kv, STRIDE, 4, 16,
                                b["kept"], STRIDE, b["counts"])
        ctx.gather_kv_pages_q8(self.pages, b["table"], width, b["kept"], b["counts"], STRIDE, n,
                               b["target"], width, b["weights"], STRIDE, b["moved"])
        t["lengths"].copy_(t["counts"])
        t["weights"].copy_(t["moved"])
        t["table"].copy_(t["target"])
        t["gl"].zero_()

    def held(self):
        """The pages as the device has them."""
        out = po.Pages.__new__(po.Pages)
        out.__dict__.update(self.cache.__dict__)
        host = self.host("keys", "values", "ks", "vs")
        out.codes = {"key": host["keys"], "value": np.empty_like(host["keys"])}
        out.set_device_values(host["values"])
        out.scales = {"key": host["ks"], "value": host["vs"]}
        return out

    def host(self, *names):
        return {n: self.t[n].cpu().numpy() for n in names}


def check_step(server, before, i):
    x = server.host("table", "lengths", "q", "g", "out", "weights", "logits", "uniform", "tokens",
                    "share", "temperature", "logprob", "rank", "entropy", "top", "top_logprob")
    held, n, heads = server.held(), len(x["lengths"]), server.heads
    lengths = x["lengths"].astype(np.int64)
    np.testing.assert_array_equal(lengths, before["lengths"] + 1)
    batch = (x["table"], np.arange(n + 1), lengths, n, 1, 1 << 20)
    want, size, score = po.attention(held, x["q"], batch, heads, x["g"])
    tol = po.attention_tolerance(size, want, score, held.head_dim, False)
    assert (np.abs(x["out"] - want) <= tol).all(), i
    want, tol = so.key_weights(held, x["q"], batch, heads, 0, 0.9, before["weights"], STRIDE)
    live = tol > 0
    assert live.sum() == 2 * lengths.sum()
    assert (np.abs(x["weights"] - want)[live] <= tol[live]).all(), i
    np.testing.assert_array_equal(x["weights"][~live], before["weights"][~live])
    for r in range(n):
        t = x["temperature"][r]
        token, share = po.sample(x["logits"][r], temperature=t, uniform=x["uniform"][r])
        assert x["tokens"][r] == token
        assert abs(x["share"][r] - share) <= 2.0 ** -23 * share
        found = so.logprobs(x["logits"][r], t, token, TOP)
        assert x["rank"][r] == found["rank"] and x["top"][r].tolist() == found["top_tokens"]
        assert abs(x["logprob"][r] - found["logprob"]) <= found["logprob_off"]
        assert abs(x["entropy"][r] - found["entropy"]) <= found["entropy_off"]
        off = np.abs(x["top_logprob"][r] - found["top_logprobs"])
        assert (off <= found["top_off"]).all()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("page_tokens", [16, 64])
def test_sequences_within_a_budget(hip_ctx, page_tokens, captured):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(page_tokens + captured)
    heads, kv, d, n = 8, 2, 128, 4
    lengths = np.array([330, 345, 320, 400], np.int32)
    width = STRIDE // page_tokens + 1
    shared = 320 // page_tokens
    pages = 2 * n * width + 3
    order = rng.permutation(pages).astype(np.int32)
    table, target = order[:2 * n * width].reshape(2, n, width)
    table[:, :shared] = table[0, :shared]
    cache = po.Pages(rng, pages, page_tokens, kv, d)
    stream = torch.cuda.Stream()
    ctx = kh.Context()
    ctx.set_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    ctx.begin_graph()
    with torch.cuda.stream(stream):
        server = Server(torch, ctx, rng, cache, table, target, lengths, heads)
        start = {name: x.clone() for name, x in server.t.items()}
        step, evict = server.step, server.evict
        step()  # (What libraries set up at their first call stays out of the graphs.)
        evict()
        if captured:
            graphs = []
            for work in (step, evict):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    work()
                graphs.append(graph)
            step, evict = graphs[0].replay, graphs[1].replay
        for name, x in start.items():
            server.t[name].copy_(x)
        position = lengths.copy()
        for i in range(6):
            if i == 3:
                have = server.held()
                x = server.host("weights", "lengths", "table")
                keep = np.array([100, 1 << 30, 17, 128], np.int32)
                server.t["keep"].copy_(torch.from_numpy(keep))
                evict()
                stream.synchronize()
                kept, counts = so.select_keys(x["weights"], x["lengths"], keep, STRIDE, 4, 16, STRIDE)
                got = server.host("kept", "lengths", "weights")
                np.testing.assert_array_equal(got["lengths"], counts)
                for b, count in enumerate(counts):
                    np.testing.assert_array_equal(got["kept"][b, :, :count], kept[b, :, :count])
                moved = so.gather(have, x["table"], kept, counts, STRIDE, target, x["weights"],
                                  STRIDE)
                after = server.held()
                for kind in ("key", "value"):
                    np.testing.assert_array_equal(after.codes[kind], have.codes[kind])
                    np.testing.assert_array_equal(after.scales[kind], have.scales[kind])
                some = ~np.isnan(moved)
                np.testing.assert_array_equal(got["weights"][some], moved[some])
            before = server.host("weights", "lengths")
            for name, x in (("qg", 2 * rng.standard_normal((n, heads, 2 * d))),
                            ("k", rng.standard_normal((n, kv, d))),
                            ("v", rng.standard_normal((n, kv, d))),
                            ("positions", np.tile(position, (4, 1))), ("uniform", rng.random(n))):
                server.t[name].copy_(torch.from_numpy(x))
            step()
            stream.synchronize()
            position += 1
            check_step(server, before, i)
    ctx.commit_graph()
    ctx.close()
